// Group normalisation with a following activation, channels last: x [N, S, C], G groups of D = C / G channels.
//   mean, var over the S * D elements of (n, g);  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) rstd;  z = xhat gamma + beta;  y = act(z)
//   dz = dy act'(z);  dgamma = sum dz xhat;  dbeta = sum dz;  gz = dz gamma
//   dx = rstd (gz - mean_g(gz) - xhat mean_g(gz xhat))
// The backward pass recomputes z with the forward pass's own sequence of roundings (norm_z), so it needs no y and takes the same
// side of an activation's corner as the forward pass did.
//
// Two forms.  HELD: a workgroup owns all rows of one sample for a slab of channels (whole groups) and keeps them in registers
// between the statistics and the result, so a tensor crosses the memory bus once.  STREAMED, where a slab does not fit:
// sums per chunk of rows, a fold over the chunks, and a second pass over the tensors.
#include "common.h"

namespace sv {
namespace {

constexpr int kGnMaxC = 4096;
constexpr int kHeldMaxC = 1024;  // widest slab of the held form

__device__ __forceinline__ float norm_xhat(float x, float mean, float rstd) {
#pragma clang fp contract(off)
    return (x - mean) * rstd;
}
__device__ __forceinline__ float norm_z(float xhat, float gamma, float beta) {
#pragma clang fp contract(off)
    return xhat * gamma + beta;
}

// V elements that one load or store moves (V a power of two, at most 16 bytes).
template <typename T, int V>
struct alignas(V * sizeof(T)) Piece {
    T v[V];
};

template <int V>
__device__ __forceinline__ void act_piece(float (&z)[V], int act, float alpha) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = act_apply(z[e], act, alpha);
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

struct GnArgs {
    const void* x;
    const void* dy;
    const float* gamma;
    const float* beta;
    float* mean;    // [N][G]: written by the forward call (may be null), read by the backward call
    float* rstd;
    void* out;      // y or dx
    float* part;    // held, backward: [N][2][C]; streamed: [N][chunks][2][C]
    float* folded;  // streamed: [N][2][C]
    float* dgamma;
    float* dbeta;
    int64_t N, S;
    int64_t rows;   // streamed: rows of a chunk
    int C, G, D, CB, slabs, chunks, act, accumulate, red;
    float eps, alpha;
};

// Workgroup -> (sample, slab).  Consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its own; the slabs of a
// sample share cache lines where a slab's row is shorter than one, so with enough samples they are dealt to one XCD.
constexpr int kXcds = 8;
__device__ __forceinline__ bool unit_of(const GnArgs& a, int64_t& n, int& slab) {
    if (a.N >= 8 * kXcds && a.slabs > 1) {
        const int64_t i = blockIdx.x / kXcds;
        n = i / a.slabs * kXcds + blockIdx.x % kXcds;
        slab = (int)(i % a.slabs);
        return n < a.N;
    }
    n = blockIdx.x / a.slabs;
    slab = (int)(blockIdx.x % a.slabs);
    return true;
}
inline int64_t held_grid(int64_t N, int slabs) {
    return N >= 8 * kXcds && slabs > 1 ? ceil_div(N, kXcds) * kXcds * slabs : N * slabs;
}

__host__ __device__ __forceinline__ bool lanes_share(int P) { return P < 64 && (P & (P - 1)) == 0; }
// Floats of LDS that sum_channels works in: a row a wave and quantity, or one a row of the workgroup.
inline int red_floats(int P, int CB, int NT) { return lanes_share(P) ? 2 * (NT / 64) * CB : NT / P * CB; }

// acc[q][e]: a thread's sums for channel p * V + e of the slab (0 in threads without work).  Leaves in out[q * CB + c] the sums
// over the workgroup, in a fixed order, and returns behind a barrier.  The rows are added in 64 bits: a
// channel's level against its group's mean makes long sums of one sign, and values of few bits round the same way in each
// addition (seen: 3e-6 in a mean of 1023 bf16 rows with 32 bits here).
template <int V, int NQ, int NT>
__device__ __forceinline__ void sum_channels(float (&acc)[NQ][V], int P, int p, int r, int rpb, int CB, float* red, float* out) {
    const int t = threadIdx.x;
    if (lanes_share(P)) {  // lanes of one piece are P apart: a wave's rows first, without LDS
        constexpr int rows = NT / 64;
        for (int o = P; o < 64; o <<= 1)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[q][e] += __shfl_xor(acc[q][e], o, 64);
        if ((t & 63) < P)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < V; ++e) red[(q * rows + (t >> 6)) * CB + p * V + e] = acc[q][e];
        __syncthreads();
        for (int i = t; i < NQ * CB; i += NT) {
            const int q = i / CB, c = i - q * CB;
            double s = 0.0;
#pragma unroll
            for (int k = 0; k < rows; ++k) s += (double)red[(q * rows + k) * CB + c];
            out[i] = (float)s;
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            if (r < rpb)
#pragma unroll
                for (int e = 0; e < V; ++e) red[r * CB + p * V + e] = acc[q][e];
            __syncthreads();
            for (int c = t; c < CB; c += NT) {
                double s = 0.0;
                for (int k = 0; k < rpb; ++k) s += (double)red[k * CB + c];
                out[q * CB + c] = (float)s;
            }
            __syncthreads();
        }
    }
}

// out[g] = sum over the D values of group g of in[g * D ..] (times w[..] where given), one wave a group.
template <int NT>
__device__ __forceinline__ void sum_groups(const float* in, const float* w, float* out, int groups, int D) {
    for (int g = threadIdx.x >> 6; g < groups; g += NT / 64) {
        double s = 0.0;
        for (int d = threadIdx.x & 63; d < D; d += 64) s += (double)in[g * D + d] * (w == nullptr ? 1.0 : (double)w[g * D + d]);
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if ((threadIdx.x & 63) == 0) out[g] = (float)s;
    }
}

// ------------------------------------------------------------------------------------------------ held
// NT threads hold K pieces each: rows r, r + rpb, ... of piece p, rpb = NT / P rows at a time, P = CB / V pieces a row.
// LDS: [a.red] partial sums | [2 * CB] channel sums | [2 * CB] group values
template <typename T, int V, int K, int NT>
__global__ __launch_bounds__(NT) void gn_fwd_held_k(GnArgs a) {
    extern __shared__ float sm[];
    float *red = sm, *ch = sm + a.red, *gv = ch + 2 * a.CB;
    int64_t n;
    int slab;
    if (!unit_of(a, n, slab)) return;
    const int c0 = slab * a.CB, CB = a.CB, P = CB / V, rpb = NT / P;
    const int p = threadIdx.x % P, r = threadIdx.x / P;
    const bool on = r < rpb && c0 + p * V < a.C;
    const int S = (int)a.S, groups = (CB < a.C - c0 ? CB : a.C - c0) / a.D;
    const int64_t base = n * a.S * a.C + c0 + p * V;
    const T* x = (const T*)a.x + base;
    Piece<T, V> buf[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int row = r + k * rpb;
        if (on && row < S) buf[k] = *(const Piece<T, V>*)(x + (int64_t)row * a.C);
    }
    float acc[1][V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[0][e] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[0][e] += (float)buf[k].v[e];
    sum_channels<V, 1, NT>(acc, P, p, r, rpb, CB, red, ch);
    sum_groups<NT>(ch, nullptr, gv, groups, a.D);
    __syncthreads();
    const float inv = 1.f / ((float)S * (float)a.D);
    // squares about that mean, and what it was off by
    float mu[V], d2[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        mu[e] = on ? gv[(p * V + e) / a.D] * inv : 0.f;
        d2[0][e] = d2[1][e] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (float)buf[k].v[e] - mu[e];
                d2[0][e] += d;
                d2[1][e] = fmaf(d, d, d2[1][e]);
            }
    sum_channels<V, 2, NT>(d2, P, p, r, rpb, CB, red, ch);
    float *s1 = gv + CB, *s2 = red;  // red is free again
    sum_groups<NT>(ch, nullptr, s1, groups, a.D);
    sum_groups<NT>(ch + CB, nullptr, s2, groups, a.D);
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += NT) {
        const float off = s1[g] * inv, var = s2[g] * inv - off * off;
        const float mean = gv[g] * inv + off;
        const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
        ch[g] = mean;
        ch[CB + g] = rstd;
        if (a.mean != nullptr) {
            a.mean[n * a.G + c0 / a.D + g] = mean;
            a.rstd[n * a.G + c0 / a.D + g] = rstd;
        }
    }
    __syncthreads();
    if (!on) return;
    float rs[V], ga[V], be[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = p * V + e, g = c / a.D;
        mu[e] = ch[g];
        rs[e] = ch[CB + g];
        ga[e] = a.gamma[c0 + c];
        be[e] = a.beta[c0 + c];
    }
    T* y = (T*)a.out + base;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int row = r + k * rpb;
        if (row < S) {
            float z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = norm_z(norm_xhat((float)buf[k].v[e], mu[e], rs[e]), ga[e], be[e]);
            act_piece<V>(z, a.act, a.alpha);
            Piece<T, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) o.v[e] = (T)z[e];
            *(Piece<T, V>*)(y + (int64_t)row * a.C) = o;
        }
    }
}

template <typename T, int V, int K, int NT>
__global__ __launch_bounds__(NT) void gn_bwd_held_k(GnArgs a) {
    extern __shared__ float sm[];
    float *red = sm, *ch = sm + a.red, *gv = ch + 2 * a.CB;
    int64_t n;
    int slab;
    if (!unit_of(a, n, slab)) return;
    const int c0 = slab * a.CB, CB = a.CB, P = CB / V, rpb = NT / P;
    const int p = threadIdx.x % P, r = threadIdx.x / P;
    const bool on = r < rpb && c0 + p * V < a.C;
    const int S = (int)a.S, groups = (CB < a.C - c0 ? CB : a.C - c0) / a.D;
    const int64_t base = n * a.S * a.C + c0 + p * V;
    const T *x = (const T*)a.x + base, *dy = (const T*)a.dy + base;
    Piece<T, V> bx[K], bg[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int row = r + k * rpb;
        if (on && row < S) {
            bx[k] = *(const Piece<T, V>*)(x + (int64_t)row * a.C);
            bg[k] = *(const Piece<T, V>*)(dy + (int64_t)row * a.C);
        }
    }
    float mu[V], rs[V], ga[V], be[V], acc[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = c0 + p * V + e, g = c / a.D;
        mu[e] = on ? a.mean[n * a.G + g] : 0.f;
        rs[e] = on ? a.rstd[n * a.G + g] : 0.f;
        ga[e] = on ? a.gamma[c] : 0.f;
        be[e] = on ? a.beta[c] : 0.f;
        acc[0][e] = acc[1][e] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = norm_xhat((float)bx[k].v[e], mu[e], rs[e]);
                const float dz = (float)bg[k].v[e] * act_slope(norm_z(xh, ga[e], be[e]), a.act, a.alpha);
                acc[0][e] += dz;
                acc[1][e] = fmaf(dz, xh, acc[1][e]);
            }
    sum_channels<V, 2, NT>(acc, P, p, r, rpb, CB, red, ch);
    for (int i = threadIdx.x; i < 2 * CB; i += NT) {
        const int q = i / CB, c = i - q * CB;
        if (c0 + c < a.C) a.part[(n * 2 + q) * a.C + c0 + c] = ch[i];
    }
    sum_groups<NT>(ch, a.gamma + c0, gv, groups, a.D);
    sum_groups<NT>(ch + CB, a.gamma + c0, gv + CB, groups, a.D);
    __syncthreads();
    if (!on) return;
    const float inv = 1.f / ((float)S * (float)a.D);
    float c1[V], c2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = (p * V + e) / a.D;
        c1[e] = gv[g] * inv;
        c2[e] = gv[CB + g] * inv;
    }
    T* dx = (T*)a.out + base;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int row = r + k * rpb;
        if (row < S) {
            Piece<T, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = norm_xhat((float)bx[k].v[e], mu[e], rs[e]);
                const float dz = (float)bg[k].v[e] * act_slope(norm_z(xh, ga[e], be[e]), a.act, a.alpha);
                o.v[e] = (T)(rs[e] * (dz * ga[e] - c1[e] - xh * c2[e]));
            }
            *(Piece<T, V>*)(dx + (int64_t)row * a.C) = o;
        }
    }
}

// ------------------------------------------------------------------------------------------------ streamed
// Workgroup -> (sample, chunk of rows, slab of channels); 256 threads, P = CB / V <= 256 pieces a row.
constexpr int kStreamThreads = 256;

// Per chunk and channel.  Forward: mean and sum of squared deviations (about the chunk's first row, then moved to the mean).
// Backward: sum dz, sum dz xhat.
template <typename T, int V, bool BWD>
__global__ __launch_bounds__(kStreamThreads) void gn_sums_k(GnArgs a) {
    extern __shared__ float sm[];
    constexpr int NT = kStreamThreads;
    const int slab = (int)(blockIdx.x % a.slabs);
    const int64_t i = blockIdx.x / a.slabs, n = i / a.chunks, chunk = i % a.chunks;
    const int c0 = slab * a.CB, CB = a.CB, P = CB / V, rpb = NT / P;
    const int p = threadIdx.x % P, r = threadIdx.x / P;
    const bool on = r < rpb && c0 + p * V < a.C;
    const int64_t r0 = chunk * a.rows, r1 = r0 + a.rows < a.S ? r0 + a.rows : a.S;
    const int64_t base = n * a.S * a.C + c0 + p * V;
    const T *x = (const T*)a.x + base, *dy = (const T*)a.dy + base;
    float acc[2][V], mu[V], rs[V], ga[V], be[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[0][e] = acc[1][e] = 0.f;
    if (on) {
        if (BWD) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = c0 + p * V + e, g = c / a.D;
                mu[e] = a.mean[n * a.G + g];
                rs[e] = a.rstd[n * a.G + g];
                ga[e] = a.gamma[c];
                be[e] = a.beta[c];
            }
        } else {
            const Piece<T, V> first = *(const Piece<T, V>*)(x + r0 * a.C);
#pragma unroll
            for (int e = 0; e < V; ++e) mu[e] = (float)first.v[e];
        }
#pragma unroll 4
        for (int64_t row = r0 + r; row < r1; row += rpb) {
            const Piece<T, V> bx = *(const Piece<T, V>*)(x + row * a.C);
            if (BWD) {
                const Piece<T, V> bg = *(const Piece<T, V>*)(dy + row * a.C);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = norm_xhat((float)bx.v[e], mu[e], rs[e]);
                    const float dz = (float)bg.v[e] * act_slope(norm_z(xh, ga[e], be[e]), a.act, a.alpha);
                    acc[0][e] += dz;
                    acc[1][e] = fmaf(dz, xh, acc[1][e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float d = (float)bx.v[e] - mu[e];
                    acc[0][e] += d;
                    acc[1][e] = fmaf(d, d, acc[1][e]);
                }
            }
        }
    }
    float *red = sm, *ch = sm + a.red;
    sum_channels<V, 2, NT>(acc, P, p, r, rpb, CB, red, ch);
    float* part = a.part + i * 2 * a.C + c0;
    for (int c = threadIdx.x; c < CB && c0 + c < a.C; c += NT) {
        float s = ch[c], q = ch[CB + c];
        if (!BWD) {
            const float m = s / (float)(r1 - r0), m2 = q - s * m;
            s = (float)((const T*)a.x)[n * a.S * a.C + r0 * a.C + c0 + c] + m;
            q = m2 < 0.f ? 0.f : m2;
        }
        part[c] = s;
        part[a.C + c] = q;
    }
}

// The chunks of a sample together, 64 channels a workgroup of 16 waves: folded[n][2][C] = the sample's mean and sum of squared
// deviations (forward) or sums (backward) per channel.
template <bool BWD>
__global__ __launch_bounds__(1024) void gn_fold_k(GnArgs a) {
    __shared__ double red[2][16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t n = blockIdx.x;
    const int c = blockIdx.y * 64 + lane;
    const float* part = a.part + n * a.chunks * 2 * a.C + c;
    const double piv = !BWD && c < a.C ? (double)part[0] : 0.0;
    double s = 0.0, q = 0.0;
    if (c < a.C) {
#pragma unroll 4
        for (int64_t k = w; k < a.chunks; k += 16) {
            const double u = (double)part[k * 2 * a.C], v = (double)part[k * 2 * a.C + a.C];
            if (BWD) {
                s += u;
                q += v;
            } else {
                const double rows = (double)((k + 1) * a.rows < a.S ? a.rows : a.S - k * a.rows), d = u - piv;
                s += rows * d;
                q += v + rows * d * d;
            }
        }
    }
    red[0][w][lane] = s;
    red[1][w][lane] = q;
    __syncthreads();
    if (w != 0 || c >= a.C) return;
    for (int k = 1; k < 16; ++k) {
        s += red[0][k][lane];
        q += red[1][k][lane];
    }
    if (!BWD) {
        const double m = s / (double)a.S, m2 = q - s * m;
        s = piv + m;
        q = m2 < 0.0 ? 0.0 : m2;
    }
    a.folded[n * 2 * a.C + c] = (float)s;
    a.folded[n * 2 * a.C + a.C + c] = (float)q;
}

// The two values of a group from its channels' folded ones, summed by one lane (D < 32) or by the 64 of a wave (`lanes`).
// Forward: mean, rstd.  Backward: mean_g(gz), mean_g(gz xhat).
template <bool BWD>
__device__ __forceinline__ void group_values(const GnArgs& a, const float* f, int g, int lane, int lanes, float& u, float& v) {
    double s = 0.0, q = 0.0;
    const double piv = BWD ? 0.0 : (double)f[g * a.D];
    for (int c = g * a.D + lane; c < (g + 1) * a.D; c += lanes) {
        if (BWD) {
            const double w = (double)a.gamma[c];
            s += w * (double)f[c];
            q += w * (double)f[a.C + c];
        } else {
            const double d = (double)f[c] - piv;
            s += d;
            q += (double)f[a.C + c] + (double)a.S * d * d;
        }
    }
    if (lanes == 64)
        for (int o = 32; o > 0; o >>= 1) {
            s += __shfl_xor(s, o, 64);
            q += __shfl_xor(q, o, 64);
        }
    const double count = (double)a.S * (double)a.D;
    if (BWD) {
        u = (float)(s / count);
        v = (float)(q / count);
    } else {
        const double m = s / (double)a.D, m2 = q - (double)a.S * s * m;
        u = (float)(piv + m);
        v = (float)(1.0 / sqrt((m2 < 0.0 ? 0.0 : m2) / count + (double)a.eps));
    }
}

template <typename T, int V, bool BWD>
__global__ __launch_bounds__(kStreamThreads) void gn_apply_k(GnArgs a) {
    extern __shared__ float gv[];  // [2][groups that the slab touches]
    constexpr int NT = kStreamThreads;
    const int64_t main = a.N * a.chunks * a.slabs;
    if (BWD && blockIdx.x >= main) {  // the last workgroups: dgamma, dbeta
        const int c = (int)(blockIdx.x - main) * NT + threadIdx.x;
        if (c >= a.C) return;
        double s = 0.0, q = 0.0;
#pragma unroll 8
        for (int64_t n = 0; n < a.N; ++n) {
            s += (double)a.folded[n * 2 * a.C + c];
            q += (double)a.folded[n * 2 * a.C + a.C + c];
        }
        a.dgamma[c] = (a.accumulate ? a.dgamma[c] : 0.f) + (float)q;
        a.dbeta[c] = (a.accumulate ? a.dbeta[c] : 0.f) + (float)s;
        return;
    }
    // last chunk first: what the statistics pass read last is what the caches still hold
    const int64_t bid = main - 1 - blockIdx.x;
    const int slab = (int)(bid % a.slabs);
    const int64_t i = bid / a.slabs, n = i / a.chunks, chunk = i % a.chunks;
    const int c0 = slab * a.CB, P = a.CB / V, rpb = NT / P;
    const int c1 = c0 + a.CB < a.C ? c0 + a.CB : a.C;
    const int g0 = c0 / a.D, g1 = (c1 - 1) / a.D + 1, gs = g1 - g0;
    const float* f = a.folded + n * 2 * a.C;
    const int lanes = a.D < 32 ? 1 : 64;
    for (int g = g0 + threadIdx.x / lanes; g < g1; g += NT / lanes) {
        float u, v;
        group_values<BWD>(a, f, g, threadIdx.x % lanes, lanes, u, v);
        if (threadIdx.x % lanes == 0) {
            gv[g - g0] = u;
            gv[gs + g - g0] = v;
            if (!BWD && chunk == 0 && a.mean != nullptr) {
                a.mean[n * a.G + g] = u;
                a.rstd[n * a.G + g] = v;
            }
        }
    }
    __syncthreads();
    const int p = threadIdx.x % P, r = threadIdx.x / P;
    if (r >= rpb || c0 + p * V >= a.C) return;
    const int64_t r0 = chunk * a.rows, r1 = r0 + a.rows < a.S ? r0 + a.rows : a.S;
    const int64_t base = n * a.S * a.C + c0 + p * V;
    const T *x = (const T*)a.x + base, *dy = (const T*)a.dy + base;
    T* out = (T*)a.out + base;
    float mu[V], rs[V], ga[V], be[V], k1[V], k2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = c0 + p * V + e, g = c / a.D;
        ga[e] = a.gamma[c];
        be[e] = a.beta[c];
        mu[e] = BWD ? a.mean[n * a.G + g] : gv[g - g0];
        rs[e] = BWD ? a.rstd[n * a.G + g] : gv[gs + g - g0];
        k1[e] = BWD ? gv[g - g0] : 0.f;
        k2[e] = BWD ? gv[gs + g - g0] : 0.f;
    }
#pragma unroll 4
    for (int64_t row = r0 + r; row < r1; row += rpb) {
        const Piece<T, V> bx = *(const Piece<T, V>*)(x + row * a.C);
        Piece<T, V> o;
        if (BWD) {
            const Piece<T, V> bg = *(const Piece<T, V>*)(dy + row * a.C);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = norm_xhat((float)bx.v[e], mu[e], rs[e]);
                const float dz = (float)bg.v[e] * act_slope(norm_z(xh, ga[e], be[e]), a.act, a.alpha);
                o.v[e] = (T)(rs[e] * (dz * ga[e] - k1[e] - xh * k2[e]));
            }
        } else {
            float z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = norm_z(norm_xhat((float)bx.v[e], mu[e], rs[e]), ga[e], be[e]);
            act_piece<V>(z, a.act, a.alpha);
#pragma unroll
            for (int e = 0; e < V; ++e) o.v[e] = (T)z[e];
        }
        *(Piece<T, V>*)(out + row * a.C) = o;
    }
}

// dgamma[c] (+)= sum over samples of part[n][1][c], dbeta[c] (+)= part[n][0][c], in a fixed order.
__global__ __launch_bounds__(1024) void gn_param_fold_k(const float* __restrict__ part, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta, int64_t parts, int C, int accumulate) {
    __shared__ float red[2][16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    float a = 0.f, b = 0.f;
    if (c < C)
#pragma unroll 8
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

// ------------------------------------------------------------------------------------------------ choice of form
struct GnPlan {
    int V, K, NT, CB, slabs;  // K = 0: streamed
    int64_t rows;
    int chunks;
};

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Largest piece (at most 16 bytes) that divides a row and that every pointer is aligned to.
int piece_of(int C, int size, uintptr_t bits) {
    int v = 16 / size;
    while (v > 1 && (C % v != 0 || bits % ((uintptr_t)v * size) != 0)) v >>= 1;
    return v;
}

// Chunks of the streamed form: about 2048 workgroups in all (8 for each CU), at least 8 rows a thread.
void plan_streamed(GnPlan& q, int64_t N, int64_t S, int C) {
    const int P = C / q.V < kStreamThreads ? C / q.V : kStreamThreads;
    q.K = 0;
    q.NT = kStreamThreads;
    q.CB = P * q.V;
    q.slabs = (int)ceil_div(C, q.CB);
    const int64_t least = 8 * (kStreamThreads / P);
    int64_t chunks = ceil_div(2048, N * q.slabs);
    if (chunks > ceil_div(S, least)) chunks = ceil_div(S, least);
    q.rows = ceil_div(S, chunks);
    q.chunks = (int)ceil_div(S, q.rows);
}

// Held where a slab of whole groups fits the registers of a workgroup: rows of about 128 bytes, else the narrowest.
// most: pieces a thread can hold.
GnPlan gn_plan(int64_t N, int64_t S, int C, int G, int size, uintptr_t bits, int most) {
    GnPlan q{};
    q.V = piece_of(C, size, bits);
    const int D = C / G, unit = D / gcd(D, q.V) * q.V;  // whole groups in whole pieces
    int wide = 128 / (unit * size) * unit;
    if (wide < unit) wide = unit;
    if (wide > C) wide = C;
    const int cbs[2] = {wide, unit > C ? C : unit};
    for (int cb : cbs) {
        const int P = cb / q.V;
        if (cb > kHeldMaxC) continue;
        static const int nts[2] = {256, 1024};
        for (int nt : nts) {
            if (P > nt) continue;
            for (int k = nt == 256 ? 2 : 8; k <= most; k *= 2)
                if (S <= (int64_t)k * (nt / P)) {
                    q.K = k;
                    q.NT = nt;
                    q.CB = cb;
                    q.slabs = (int)ceil_div(C, cb);
                    return q;
                }
        }
    }
    plan_streamed(q, N, S, C);
    return q;
}

// workspace: [N][2][C] folded sums | [N][chunks][2][C] partial sums.  The chunks do not depend on the piece the alignment
// allows beyond what gn_plan_most bounds.
int64_t gn_most_chunks(int64_t N, int64_t S, int C) {
    int64_t most = 1;
    for (int v = 1; v <= 8; v *= 2)
        if (C % v == 0) {
            GnPlan q{};
            q.V = v;
            plan_streamed(q, N, S, C);
            if (q.chunks > most) most = q.chunks;
        }
    return most;
}
size_t gn_ws_bytes(int64_t N, int64_t S, int C) {
    return (size_t)N * 2 * C * (1 + (size_t)gn_most_chunks(N, S, C)) * sizeof(float);
}

int gn_check(const char* who, int64_t N, int64_t S, int C, int G, int act, void* ws, size_t ws_bytes) {
    SV_REQUIRE(N >= 0 && S > 0 && C > 0 && C <= kGnMaxC, "%s: bad extents (N=%lld S=%lld C=%d)", who, (long long)N,
               (long long)S, C);
    SV_REQUIRE(G >= 1 && C % G == 0, "%s: %d channels do not split into %d groups", who, C, G);
    SV_REQUIRE(S <= ((int64_t)1 << 40) / C && N <= ((int64_t)1 << 40) / (S * C), "%s: tensor too large", who);
    SV_REQUIRE(act >= SV_ACT_NONE && act <= SV_ACT_SIGMOID, "%s: activation %d unknown", who, act);
    if (N == 0) return SV_OK;
    SV_REQUIRE(N <= (1 << 24) && N * C <= 0x3fffffff, "%s: too many samples", who);
    const size_t need = gn_ws_bytes(N, S, C);
    if (ws == nullptr || ws_bytes < need) return fail(SV_E_WORKSPACE, "%s: workspace %zu bytes < required %zu", who, ws_bytes, need);
    return SV_OK;
}

// f(integral_constant...) with T, V as template arguments
#define SV_GN_V(T, v, BODY)                                                    \
    switch (v) {                                                               \
        case 8: if constexpr (sizeof(T) == 2) { constexpr int V = 8; BODY } break; \
        case 4: { constexpr int V = 4; BODY } break;                           \
        case 2: { constexpr int V = 2; BODY } break;                           \
        default: { constexpr int V = 1; BODY } break;                          \
    }

template <typename T, bool BWD>
void launch_held(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    const dim3 grid((unsigned)held_grid(a.N, q.slabs));
    const size_t lds = ((size_t)a.red + 4 * (size_t)q.CB) * sizeof(float);  // at most 48 KB

#define SV_GN_GO(K, NT)                                                                                   \
    do {                                                                                                  \
        if constexpr (BWD) hipLaunchKernelGGL((gn_bwd_held_k<T, V, K, NT>), grid, dim3(NT), lds, st, a);  \
        else hipLaunchKernelGGL((gn_fwd_held_k<T, V, K, NT>), grid, dim3(NT), lds, st, a);                \
    } while (0)
    SV_GN_V(T, q.V,
        if (q.NT == 256) {
            if (q.K == 2) SV_GN_GO(2, 256);
            else if (q.K == 4) SV_GN_GO(4, 256);
            else if (q.K == 8) SV_GN_GO(8, 256);
            else if constexpr (!BWD) SV_GN_GO(16, 256);
        } else {
            if (q.K == 8) SV_GN_GO(8, 1024);
            else if constexpr (!BWD) SV_GN_GO(16, 1024);
        }
    )
#undef SV_GN_GO
}

template <typename T, bool BWD>
void launch_streamed(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    const int64_t main = a.N * q.chunks * q.slabs;
    const size_t lds = ((size_t)a.red + 2 * (size_t)q.CB) * sizeof(float);  // at most 24 KB
    const size_t lds_apply = 2 * ((size_t)q.CB / a.D + 2) * sizeof(float);
    SV_GN_V(T, q.V,
        hipLaunchKernelGGL((gn_sums_k<T, V, BWD>), dim3((unsigned)main), dim3(kStreamThreads), lds, st, a);
        hipLaunchKernelGGL((gn_fold_k<BWD>), dim3((unsigned)a.N, (unsigned)ceil_div(a.C, 64)), dim3(1024), 0, st, a);
        hipLaunchKernelGGL((gn_apply_k<T, V, BWD>), dim3((unsigned)(main + (BWD ? ceil_div(a.C, kStreamThreads) : 0))),
                           dim3(kStreamThreads), lds_apply, st, a);
    )
}

template <typename T, bool BWD>
void launch(GnArgs& a, void* workspace, hipStream_t st) {
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)a.dy;
    // a backward thread holds two tensors: 8 pieces of each
    const GnPlan q = gn_plan(a.N, a.S, a.C, a.G, sizeof(T), bits, BWD ? 8 : 16);
    a.CB = q.CB;
    a.red = red_floats(q.CB / q.V, q.CB, q.NT);
    a.slabs = q.slabs;
    a.rows = q.rows;
    a.chunks = q.chunks;
    a.folded = (float*)workspace;
    if (q.K > 0) {
        a.part = (float*)workspace;
        launch_held<T, BWD>(a, q, st);
        if (BWD)
            hipLaunchKernelGGL(gn_param_fold_k, dim3((unsigned)ceil_div(a.C, 64)), dim3(1024), 0, st, a.part, a.dgamma, a.dbeta,
                               a.N, a.C, a.accumulate);
    } else {
        a.part = a.folded + a.N * 2 * a.C;
        launch_streamed<T, BWD>(a, q, st);
    }
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" {

size_t sv_groupnorm_workspace_bytes(int64_t N, int64_t S, int C, int groups) {
    if (N <= 0 || S <= 0 || C <= 0 || C > kGnMaxC || groups < 1 || C % groups) return 0;
    return gn_ws_bytes(N, S, C);
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
    GnArgs a{};
    a.x = x;
    a.gamma = gamma;
    a.beta = beta;
    a.out = y;
    a.mean = save_mean;
    a.rstd = save_rstd;
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = groups;
    a.D = C / groups;
    a.eps = eps;
    a.act = act;
    a.alpha = alpha;
    if (dtype == SV_F32) launch<float, false>(a, workspace, to_stream(stream));
    else launch<__bf16, false>(a, workspace, to_stream(stream));
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
    if (N == 0) {
        hipLaunchKernelGGL(gn_param_fold_k, dim3((unsigned)ceil_div(C, 64)), dim3(1024), 0, st, nullptr, dgamma, dbeta, (int64_t)0, C,
                           accumulate);
        return check_launch("sv_groupnorm_act_bwd");
    }
    SV_REQUIRE(x && dy && gamma && beta && save_mean && save_rstd && dx, "sv_groupnorm_act_bwd: null tensor");
    GnArgs a{};
    a.x = x;
    a.dy = dy;
    a.gamma = gamma;
    a.beta = beta;
    a.mean = const_cast<float*>(save_mean);
    a.rstd = const_cast<float*>(save_rstd);
    a.out = dx;
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.accumulate = accumulate;
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = groups;
    a.D = C / groups;
    a.act = act;
    a.alpha = alpha;
    if (dtype == SV_F32) launch<float, true>(a, workspace, st);
    else launch<__bf16, true>(a, workspace, st);
    return check_launch("sv_groupnorm_act_bwd");
}

}  // extern "C"
