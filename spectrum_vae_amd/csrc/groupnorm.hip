// Group normalisation with a following activation, channels last: x [N, S, C], G groups of D = C / G channels.
//   mean, var over the S * D elements of (n, g);  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) rstd;  z = xhat gamma + beta;  y = act(z)
//   dz = dy act'(z);  dgamma = sum dz xhat;  dbeta = sum dz;  gz = dz gamma
//   dx = rstd (gz - mean_g(gz) - xhat mean_g(gz xhat))
// The backward pass recomputes z with the forward pass's own sequence of roundings (norm_z), so it needs no y and takes the same
// side of an activation's corner as the forward pass did.
#include "common.h"

namespace sv {
namespace {

constexpr int kGnMaxC = 4096;
constexpr int kGnMaxChunks = 4096;

// Rows of a sample are cut into `chunks` equal parts, one workgroup each.
struct GnPlan {
    int64_t rows;  // rows of a chunk (the last may have fewer)
    int chunks;
};
inline GnPlan gn_plan(int64_t N, int64_t S, int C) {
    const int64_t rif = C < 256 ? 256 / C : 1;
    int64_t rows = 16 * rif;  // 16 rows a thread at least
    const int64_t want = ceil_div(N * S, (int64_t)4096);
    if (rows < want) rows = want;
    if (rows < ceil_div(S, (int64_t)kGnMaxChunks)) rows = ceil_div(S, (int64_t)kGnMaxChunks);
    if (rows > S) rows = S;
    return {rows, (int)ceil_div(S, rows)};
}

__device__ __forceinline__ float norm_xhat(float x, float mean, float rstd) {
#pragma clang fp contract(off)
    return (x - mean) * rstd;
}
__device__ __forceinline__ float norm_z(float xhat, float gamma, float beta) {
#pragma clang fp contract(off)
    return xhat * gamma + beta;
}
// d act / d z from z; at 0 the slope of the negative side.
__device__ __forceinline__ float act_slope(float z, int act, float alpha) {
    switch (act) {
        case SV_ACT_RELU: return z > 0.f ? 1.f : 0.f;
        case SV_ACT_ELU: return z > 0.f ? 1.f : __expf(z);
        case SV_ACT_LRELU: return z > 0.f ? 1.f : alpha;
        case SV_ACT_TANH: { const float t = fast_tanh(z); return 1.f - t * t; }
        case SV_ACT_SIGMOID: { const float y = __builtin_amdgcn_rcpf(1.f + __expf(-z)); return y * (1.f - y); }
        default: return 1.f;
    }
}

// Per chunk and channel: mean and sum of squared deviations about it -> part[chunk][2][C].  A thread sums about its first
// value; the threads' sums are then combined about their common mean.
template <typename T>
__global__ __launch_bounds__(256) void gn_stats_k(const T* __restrict__ x, float* __restrict__ part, int64_t S, int C,
                                                   GnPlan p) {
    __shared__ float s_n[256], s_mean[256], s_m2[256];
    const int64_t n = blockIdx.x / p.chunks;
    const int ch = (int)(blockIdx.x % p.chunks);
    const int64_t r0 = ch * p.rows, r1 = r0 + p.rows < S ? r0 + p.rows : S;
    x += n * S * C;
    part += (int64_t)blockIdx.x * 2 * C;
    const int cw = C < 256 ? C : 256, rif = 256 / cw;
    const int cl = threadIdx.x % cw, rr = threadIdx.x / cw;
    for (int c0 = 0; c0 < C; c0 += cw) {
        const int c = c0 + cl;
        float cnt = 0.f, s = 0.f, q = 0.f, piv = 0.f;
        if (rr < rif && c < C && r0 + rr < r1) {
            piv = (float)x[(r0 + rr) * C + c];
            for (int64_t r = r0 + rr; r < r1; r += rif) {
                const float d = (float)x[r * C + c] - piv;
                s += d;
                q = fmaf(d, d, q);
                cnt += 1.f;
            }
        }
        const float m = cnt > 0.f ? s / cnt : 0.f;
        s_n[threadIdx.x] = cnt;
        s_mean[threadIdx.x] = piv + m;
        const float m2 = q - s * m;
        s_m2[threadIdx.x] = m2 < 0.f ? 0.f : m2;  // NaN stays
        __syncthreads();
        if (rr == 0 && c < C) {
            float tn = 0.f, tm = 0.f, t2 = 0.f;
            for (int k = 0; k < rif; ++k) {
                const int i = k * cw + cl;
                if (s_n[i] == 0.f) continue;
                const float nn = tn + s_n[i], d = s_mean[i] - tm;
                tm += d * (s_n[i] / nn);
                t2 += s_m2[i] + d * d * (tn * s_n[i] / nn);
                tn = nn;
            }
            part[c] = tm;
            part[C + c] = t2;
        }
        __syncthreads();
    }
}

// One wave per (n, g): the chunks' per-channel moments -> mean, rstd of the group, in f64.
__global__ __launch_bounds__(64) void gn_fold_stats_k(const float* __restrict__ part, float* __restrict__ mean,
                                                       float* __restrict__ rstd, int64_t S, int C, int G, float eps, GnPlan p) {
    const int64_t n = blockIdx.x / G;
    const int g = (int)(blockIdx.x % G), D = C / G;
    part += n * p.chunks * 2 * C + g * D;
    const int64_t items = (int64_t)p.chunks * D;
    const double count = (double)S * D;
    double s = 0.0, q = 0.0;
    for (int64_t i = threadIdx.x; i < items; i += 64) {
        const int64_t ch = i / D, d = i % D;
        const double rows = (double)((ch + 1) * p.rows < S ? p.rows : S - ch * p.rows);
        s += rows * (double)part[ch * 2 * C + d];
    }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    const double mu = s / count;
    for (int64_t i = threadIdx.x; i < items; i += 64) {
        const int64_t ch = i / D, d = i % D;
        const double rows = (double)((ch + 1) * p.rows < S ? p.rows : S - ch * p.rows);
        const double dm = (double)part[ch * 2 * C + d] - mu;
        q += (double)part[ch * 2 * C + C + d] + rows * dm * dm;
    }
    for (int o = 32; o > 0; o >>= 1) q += __shfl_xor(q, o, 64);
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = (float)mu;
        rstd[blockIdx.x] = (float)(1.0 / sqrt(q / count + (double)eps));
    }
}

template <typename T>
__global__ __launch_bounds__(256) void gn_apply_k(const T* __restrict__ x, const float* __restrict__ gamma,
                                                   const float* __restrict__ beta, const float* __restrict__ mean,
                                                   const float* __restrict__ rstd, T* __restrict__ y, int64_t total,
                                                   int64_t SC, int C, int G, int act, float alpha) {
    const int D = C / G;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int c = (int)(i % C);
        const int64_t g = (i / SC) * G + c / D;
        y[i] = (T)act_apply(norm_z(norm_xhat((float)x[i], mean[g], rstd[g]), gamma[c], beta[c]), act, alpha);
    }
}

// Per chunk and channel: sum dz, sum dz xhat -> part[chunk][2][C].
template <typename T>
__global__ __launch_bounds__(256) void gn_bwd_sums_k(const T* __restrict__ x, const T* __restrict__ dy,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      float* __restrict__ part, int64_t S, int C, int G, int act,
                                                      float alpha, GnPlan p) {
    __shared__ float s_a[256], s_b[256];
    const int64_t n = blockIdx.x / p.chunks;
    const int ch = (int)(blockIdx.x % p.chunks), D = C / G;
    const int64_t r0 = ch * p.rows, r1 = r0 + p.rows < S ? r0 + p.rows : S;
    x += n * S * C;
    dy += n * S * C;
    part += (int64_t)blockIdx.x * 2 * C;
    const int cw = C < 256 ? C : 256, rif = 256 / cw;
    const int cl = threadIdx.x % cw, rr = threadIdx.x / cw;
    for (int c0 = 0; c0 < C; c0 += cw) {
        const int c = c0 + cl;
        float a = 0.f, b = 0.f;
        if (rr < rif && c < C) {
            const float mu = mean[n * G + c / D], rs = rstd[n * G + c / D], ga = gamma[c], be = beta[c];
            for (int64_t r = r0 + rr; r < r1; r += rif) {
                const float xh = norm_xhat((float)x[r * C + c], mu, rs);
                const float dz = (float)dy[r * C + c] * act_slope(norm_z(xh, ga, be), act, alpha);
                a += dz;
                b = fmaf(dz, xh, b);
            }
        }
        s_a[threadIdx.x] = a;
        s_b[threadIdx.x] = b;
        __syncthreads();
        if (rr == 0 && c < C) {
            for (int k = 1; k < rif; ++k) {
                a += s_a[k * cw + cl];
                b += s_b[k * cw + cl];
            }
            part[c] = a;
            part[C + c] = b;
        }
        __syncthreads();
    }
}

// One wave per (n, g): mean_g(gz), mean_g(gz xhat) -> coef[n][g][2].
__global__ __launch_bounds__(64) void gn_bwd_group_k(const float* __restrict__ part, const float* __restrict__ gamma,
                                                      float* __restrict__ coef, int64_t S, int C, int G, GnPlan p) {
    const int64_t n = blockIdx.x / G;
    const int g = (int)(blockIdx.x % G), D = C / G;
    part += n * p.chunks * 2 * C + g * D;
    const int64_t items = (int64_t)p.chunks * D;
    double a = 0.0, b = 0.0;
    for (int64_t i = threadIdx.x; i < items; i += 64) {
        const int64_t ch = i / D, d = i % D;
        const double ga = (double)gamma[g * D + d];
        a += ga * (double)part[ch * 2 * C + d];
        b += ga * (double)part[ch * 2 * C + C + d];
    }
    for (int o = 32; o > 0; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if (threadIdx.x == 0) {
        const double count = (double)S * D;
        coef[2 * (int64_t)blockIdx.x] = (float)(a / count);
        coef[2 * (int64_t)blockIdx.x + 1] = (float)(b / count);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void gn_bwd_apply_k(const T* __restrict__ x, const T* __restrict__ dy,
                                                       const float* __restrict__ gamma, const float* __restrict__ beta,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd,
                                                       const float* __restrict__ coef, T* __restrict__ dx, int64_t total,
                                                       int64_t SC, int C, int G, int act, float alpha) {
    const int D = C / G;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int c = (int)(i % C);
        const int64_t g = (i / SC) * G + c / D;
        const float xh = norm_xhat((float)x[i], mean[g], rstd[g]);
        const float dz = (float)dy[i] * act_slope(norm_z(xh, gamma[c], beta[c]), act, alpha);
        dx[i] = (T)(rstd[g] * (dz * gamma[c] - coef[2 * g] - xh * coef[2 * g + 1]));
    }
}

// dgamma[c] (+)= sum over parts of part[.][1][c], dbeta[c] (+)= part[.][0][c], in a fixed order.
__global__ __launch_bounds__(1024) void gn_param_fold_k(const float* __restrict__ part, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta, int64_t parts, int C, int accumulate) {
    __shared__ float red[2][16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    float a = 0.f, b = 0.f;
    if (c < C)
        for (int64_t i = w; i < parts; i += 16) {
            a += part[i * 2 * C + c];
            b += part[i * 2 * C + C + c];
        }
    red[0][w][lane] = a;
    red[1][w][lane] = b;
    __syncthreads();
    if (w != 0 || c >= C) return;
    for (int k = 1; k < 16; ++k) {
        a += red[0][k][lane];
        b += red[1][k][lane];
    }
    dgamma[c] = (accumulate ? dgamma[c] : 0.f) + b;
    dbeta[c] = (accumulate ? dbeta[c] : 0.f) + a;
}

// workspace: [N * chunks][2][C] partial sums | [N][G][2] group values (statistics or backward coefficients)
size_t gn_ws_bytes(int64_t N, int64_t S, int C, int G) {
    const GnPlan p = gn_plan(N, S, C);
    return ((size_t)N * p.chunks * 2 * C + (size_t)N * G * 2) * sizeof(float);
}

int gn_check(const char* who, int64_t N, int64_t S, int C, int G, int act, void* ws, size_t ws_bytes) {
    SV_REQUIRE(N >= 0 && S > 0 && C > 0 && C <= kGnMaxC, "%s: bad extents (N=%lld S=%lld C=%d)", who, (long long)N,
               (long long)S, C);
    SV_REQUIRE(G >= 1 && C % G == 0, "%s: %d channels do not split into %d groups", who, C, G);
    SV_REQUIRE(S <= ((int64_t)1 << 40) / C && N <= ((int64_t)1 << 40) / (S * C), "%s: tensor too large", who);
    SV_REQUIRE(act >= SV_ACT_NONE && act <= SV_ACT_SIGMOID, "%s: activation %d unknown", who, act);
    if (N == 0) return SV_OK;
    SV_REQUIRE(N * gn_plan(N, S, C).chunks <= 0x7fffffff && N * G <= 0x7fffffff, "%s: too many samples", who);
    const size_t need = gn_ws_bytes(N, S, C, G);
    if (ws == nullptr || ws_bytes < need) return fail(SV_E_WORKSPACE, "%s: workspace %zu bytes < required %zu", who, ws_bytes, need);
    return SV_OK;
}

}  // namespace

#define SV_GN_T(dtype, BODY)          \
    do {                              \
        if ((dtype) == SV_F32) {      \
            typedef float T;          \
            BODY                      \
        } else {                      \
            typedef __bf16 T;         \
            BODY                      \
        }                             \
    } while (0)

}  // namespace sv

using namespace sv;

extern "C" {

size_t sv_groupnorm_workspace_bytes(int64_t N, int64_t S, int C, int groups) {
    if (N <= 0 || S <= 0 || C <= 0 || C > kGnMaxC || groups < 1 || C % groups) return 0;
    return gn_ws_bytes(N, S, C, groups);
}

int sv_groupnorm_act_fwd(const void* x, const float* gamma, const float* beta, void* y, float* save_mean, float* save_rstd,
                         int64_t N, int64_t S, int C, int groups, float eps, int act, float alpha, void* workspace,
                         size_t workspace_bytes, int dtype, sv_stream_t stream) {
    SV_F32_OR_BF16(dtype, "sv_groupnorm_act_fwd");
    int rc = gn_check("sv_groupnorm_act_fwd", N, S, C, groups, act, workspace, workspace_bytes);
    if (rc) return rc;
    SV_REQUIRE((save_mean == nullptr) == (save_rstd == nullptr), "sv_groupnorm_act_fwd: save_mean and save_rstd go together");
    if (N == 0) return SV_OK;
    SV_REQUIRE(x && gamma && beta && y, "sv_groupnorm_act_fwd: null tensor");
    hipStream_t st = to_stream(stream);
    const GnPlan p = gn_plan(N, S, C);
    float* part = (float*)workspace;
    float* mean = save_mean ? save_mean : part + (size_t)N * p.chunks * 2 * C;
    float* rstd = save_rstd ? save_rstd : mean + N * groups;
    SV_GN_T(dtype, hipLaunchKernelGGL(gn_stats_k<T>, dim3((unsigned)(N * p.chunks)), dim3(256), 0, st, (const T*)x, part, S, C, p););
    hipLaunchKernelGGL(gn_fold_stats_k, dim3((unsigned)(N * groups)), dim3(64), 0, st, part, mean, rstd, S, C, groups, eps, p);
    SV_GN_T(dtype, hipLaunchKernelGGL(gn_apply_k<T>, dim3(ew_grid(N * S * C, 256, 16384)), dim3(256), 0, st, (const T*)x, gamma,
                                      beta, mean, rstd, (T*)y, N * S * C, S * C, C, groups, act, alpha););
    return check_launch("sv_groupnorm_act_fwd");
}

int sv_groupnorm_act_bwd(const void* x, const void* dy, const float* gamma, const float* beta, const float* save_mean,
                         const float* save_rstd, void* dx, float* dgamma, float* dbeta, int accumulate, int64_t N, int64_t S,
                         int C, int groups, int act, float alpha, void* workspace, size_t workspace_bytes, int dtype,
                         sv_stream_t stream) {
    SV_F32_OR_BF16(dtype, "sv_groupnorm_act_bwd");
    int rc = gn_check("sv_groupnorm_act_bwd", N, S, C, groups, act, workspace, workspace_bytes);
    if (rc) return rc;
    SV_REQUIRE(dgamma && dbeta, "sv_groupnorm_act_bwd: null tensor");
    hipStream_t st = to_stream(stream);
    const GnPlan p = N ? gn_plan(N, S, C) : GnPlan{1, 1};
    float* part = (float*)workspace;
    float* coef = part + (size_t)N * p.chunks * 2 * C;
    if (N > 0) {
        SV_REQUIRE(x && dy && gamma && beta && save_mean && save_rstd && dx, "sv_groupnorm_act_bwd: null tensor");
        SV_GN_T(dtype, hipLaunchKernelGGL(gn_bwd_sums_k<T>, dim3((unsigned)(N * p.chunks)), dim3(256), 0, st, (const T*)x,
                                          (const T*)dy, gamma, beta, save_mean, save_rstd, part, S, C, groups, act, alpha, p););
        hipLaunchKernelGGL(gn_bwd_group_k, dim3((unsigned)(N * groups)), dim3(64), 0, st, part, gamma, coef, S, C, groups, p);
        SV_GN_T(dtype, hipLaunchKernelGGL(gn_bwd_apply_k<T>, dim3(ew_grid(N * S * C, 256, 16384)), dim3(256), 0, st, (const T*)x,
                                          (const T*)dy, gamma, beta, save_mean, save_rstd, coef, (T*)dx, N * S * C, S * C, C,
                                          groups, act, alpha););
    }
    hipLaunchKernelGGL(gn_param_fold_k, dim3((unsigned)ceil_div(C, 64)), dim3(1024), 0, st, part, dgamma, dbeta, N * p.chunks, C,
                       accumulate);
    return check_launch("sv_groupnorm_act_bwd");
}

}  // extern "C"
