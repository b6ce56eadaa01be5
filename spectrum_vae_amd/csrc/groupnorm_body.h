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
// sums per chunk of rows, a fold over the chunks (a launch, or the start of the second pass), and a second pass over the tensors.
//
// What bounds it: the memory, 8 flops a byte at most.  A copy of 512 MB runs at 5.3 TB/s here, and a launch that does next to nothing
// takes 3.5 us.  Measured, with alternating tensors:
//   held      forward   1024 x 32x32x64 f32     537 MB moved   100 us   5.4 TB/s
//             forward   512 x 32x32x64 bf16     134 MB          32 us   4.2
//             backward  1024 x 16x16x256 bf16   403 MB          83 us   4.8   (6 us of it gn_param_fold_k)
//             forward   1 x 8x8x64 f32                         3.7 us
//             backward  64 x 8x8x128 f32          6 MB         7.2 us   two launches in a row of calls; each by itself 5.9 and 3.0
//   streamed  forward   2 x 512x512x128 bf16    268 MB          84 us   403 MB with the second reading: 4.8 TB/s
//             backward  4 x 256x256x64 f32      201 MB          64 us   336 MB with the second reading: 5.2 TB/s
//             forward   64 x 90x90x32 bf16       66 MB          27 us   two passes of 33 and 66 MB and their launches
#pragma once
#include <type_traits>

#include "common.h"

namespace sv {
namespace {

constexpr int kGnMaxC = 4096;
constexpr int kHeldMaxC = 512;                // widest slab of the held form
constexpr int kHeldSlots = 4096;              // most slots x channels of it (LDS: 32 KB, and at most 16 for the groups)
constexpr int kHeldFwd = 256, kHeldBwd = 128;  // bytes of a tensor that a thread holds, forward and (each of two) backward

__device__ __forceinline__ float norm_xhat(float x, float mean, float rstd) {
#pragma clang fp contract(off)
    return (x - mean) * rstd;
}
__device__ __forceinline__ float norm_z(float xhat, float gamma, float beta) {
#pragma clang fp contract(off)
    return xhat * gamma + beta;
}

// V elements that one load or store moves (V a power of two, at most 16 bytes), held as words: two bf16 stay in one register.
template <int BYTES> struct WordsOf { typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4))); };
template <> struct WordsOf<4> { typedef uint32_t type; };
template <> struct WordsOf<2> { typedef uint16_t type; };
template <typename T, int V> using Piece = typename WordsOf<V * (int)sizeof(T)>::type;

template <typename T, int V>
__device__ __forceinline__ float get(const Piece<T, V>& w, int e) {
    if constexpr (V * sizeof(T) == 2) return __uint_as_float((uint32_t)w << 16);
    else if constexpr (sizeof(T) == 2 && V == 2) return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    else if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else if constexpr (V == 1) return __uint_as_float(w);
    else return __uint_as_float(w[e]);
}
template <typename T, int V>
__device__ __forceinline__ Piece<T, V> put(const float (&v)[V]) {
    typedef T Elements __attribute__((ext_vector_type(V)));
    Elements o;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = (T)v[e];
    return __builtin_bit_cast(Piece<T, V>, o);
}
// The compiler forgets what it knows of a piece: values worked out from it before (bf16 widened above all) are worked out again
// instead of being kept in twice the registers.
template <typename P>
__device__ __forceinline__ void forget(P& w) {
    if constexpr (sizeof(P) >= 4) asm volatile("" : "+v"(w));
}
template <typename P>
__device__ __forceinline__ P& piece_at(const void* base, uint32_t bytes) {
    return *(P*)((char*)base + bytes);
}

template <bool FAR, typename P>
__device__ __forceinline__ P load_piece(const P& from) {
    return FAR ? __builtin_nontemporal_load(&from) : from;
}
template <bool FAR, typename P>
__device__ __forceinline__ void store_piece(P& to, P w) {
    if (FAR) __builtin_nontemporal_store(w, &to);
    else to = w;
}

// f(the activation's code as a constant): one branch ahead of a loop instead of one an element.
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
    switch (act) {
        case SV_ACT_RELU: f(std::integral_constant<int, SV_ACT_RELU>{}); break;
        case SV_ACT_ELU: f(std::integral_constant<int, SV_ACT_ELU>{}); break;
        case SV_ACT_LRELU: f(std::integral_constant<int, SV_ACT_LRELU>{}); break;
        case SV_ACT_TANH: f(std::integral_constant<int, SV_ACT_TANH>{}); break;
        case SV_ACT_SIGMOID: f(std::integral_constant<int, SV_ACT_SIGMOID>{}); break;
        default: f(std::integral_constant<int, SV_ACT_NONE>{}); break;
    }
}
// act(z).  NaN stays NaN behind every activation (act_apply's ReLU makes it 0, and one such input would turn the whole group into
// clean zeros).
__device__ __forceinline__ float act_value(float z, int act, float alpha) {
    return act == SV_ACT_RELU ? (z <= 0.f ? 0.f : z) : act_apply(z, act, alpha);
}
// d act / d z from z; at 0 the slope of the negative side (also where z is NaN and the slope has two values: see keep_nan).
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
// A channel's sums of dz and dz xhat where z was NaN and the slope did not show it: xhat did, or gamma or beta is NaN.  (Once a
// channel; a slope that is NaN for NaN is a comparison more an element, 1 to 2 % of the whole backward pass.)
__device__ __forceinline__ void keep_nan(float& dz, float& dz_xhat, float gamma, float beta, int act) {
    if (act != SV_ACT_RELU && act != SV_ACT_LRELU) return;
    if (dz_xhat != dz_xhat || gamma != gamma || beta != beta) dz = dz_xhat = __uint_as_float(0x7fc00000u);
}

// ------------------------------------------------------------------------------------------------ sums across lanes
// One vector instruction a step (data-parallel primitives inside a row of 16 lanes, lane swaps between rows), no LDS.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kRor4 = 0x124, kRor8 = 0x128, kMirror8 = 0x141, kMirror16 = 0x140;
__device__ __forceinline__ float add_row16(float v) {  // + the neighbouring row of 16
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_half32(float v) {  // + the other half of the wave
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sum over the lanes that are a multiple of P apart (P a power of two up to 64); every lane gets its sum.
__device__ __forceinline__ float sum_stride(float v, int P) {
    if (P <= 1) v = dpp_add<kXor1>(v);
    if (P <= 2) v = dpp_add<kXor2>(v);
    if (P <= 4) v = dpp_add<kRor4>(v);
    if (P <= 8) v = dpp_add<kRor8>(v);
    if (P <= 16) v = add_row16(v);
    if (P <= 32) v = add_half32(v);
    return v;
}
// Sum over aligned runs of n neighbouring lanes (n a power of two up to 64); every lane gets its run's sum.
__device__ __forceinline__ float sum_run(float v, int n) {
    if (n >= 2) v = dpp_add<kXor1>(v);
    if (n >= 4) v = dpp_add<kXor2>(v);
    if (n >= 8) v = dpp_add<kMirror8>(v);
    if (n >= 16) v = dpp_add<kMirror16>(v);
    if (n >= 32) v = add_row16(v);
    if (n >= 64) v = add_half32(v);
    return v;
}

// Lanes that share a sum of `items` terms: a power of two, at most a wave.
__device__ __forceinline__ int lanes_for(int items) {
    int l = 1;
    while (l < items && l < 64) l <<= 1;
    return l;
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
    float* folded;  // streamed: [N][2][C], the chunks joined by gn_fold_k, or
    float* groups;  //           [N][chunks][2][G], the chunks' values of whole groups, joined in the second pass (else null)
    float* dgamma;
    float* dbeta;
    int64_t N, S;
    int64_t rows;   // streamed: rows of a chunk
    int C, G, D, CB, slabs, chunks, act, accumulate;
    int P;          // pieces of a slab's row
    int log_q;      // held: threads of a row, a power of two >= P
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

// ------------------------------------------------------------------------------------------------ held
// NT threads hold K pieces each: Q = 2^log_q >= P threads a row (P pieces), rows r, r + NT / Q, ...  A wave (a row's threads where
// they are more than a wave) is a slot: its rows are summed across lanes, the slots' sums meet in LDS.
// Forward: a slot's mean and sum of squares about that mean, joined by the parts' counts (as exact as two passes over everything,
// with one barrier).  GROUPS: D is a power of two, D >= V and P = Q, so a slot sums whole groups; else it sums channels.
// FAR: nontemporal stores (1), loads and stores (2).
template <int NT>
struct Slots {
    int lanes, count, mine;  // threads of a slot, slots, this thread's
    __device__ __forceinline__ explicit Slots(int log_q) {
        lanes = log_q < 6 ? 64 : 1 << log_q;
        count = NT / lanes;
        mine = threadIdx.x / lanes;
    }
    // Rows of the sample that slot `s` holds.
    __device__ __forceinline__ float rows(int s, int S, int log_q) const {
        const int rpb = NT >> log_q, each = lanes >> log_q, rest = S % rpb - s * each;
        return (float)(S / rpb * each + (rest < 0 ? 0 : rest < each ? rest : each));
    }
};

// LDS: [2][slots][groups or channels of a slab], then [2][groups] (channels only).
// Two workgroups of 1024 fit a CU with at most 64 registers a thread, which 128 bytes of f32 leave room for.
template <typename T, int V, int K, int NT, bool GROUPS, int FAR>
__global__ __launch_bounds__(NT, (GROUPS && K * V * sizeof(T) <= 128 && sizeof(T) == 4 ? 8 : 1)) void gn_fwd_held_k(GnArgs a) {
    extern __shared__ float sm[];
    int64_t n;
    int slab;
    if (!unit_of(a, n, slab)) return;
    constexpr int NV = GROUPS ? 1 : V;  // sums a thread takes part in
    const int Q = 1 << a.log_q, rpb = NT >> a.log_q, S = (int)a.S;
    const int p = threadIdx.x & (Q - 1), r = threadIdx.x >> a.log_q;
    const int c0 = slab * a.CB + p * V, D = a.D;
    const bool on = p < a.P && c0 < a.C;
    // a slab's base for all threads, 32-bit offsets in it (a held sample has at most 16384 rows)
    const int64_t base = n * a.S * a.C + slab * a.CB;
    const uint32_t at0 = (uint32_t)(r * a.C + p * V) * sizeof(T), step = (uint32_t)(rpb * a.C) * sizeof(T);
    typedef Piece<T, V> Q_;
    const T* x = (const T*)a.x + base;
    Q_ buf[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S) buf[k] = load_piece<FAR == 2>(piece_at<const Q_>(x, at0 + k * step));
    float ga[V], be[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        ga[e] = on ? a.gamma[c0 + e] : 0.f;
        be[e] = on ? a.beta[c0 + e] : 0.f;
    }
    const Slots<NT> slot(a.log_q);
    const int run = GROUPS ? D / V : 1, width = GROUPS ? a.CB / D : a.CB, at = GROUPS ? p / run : p * V;
    float sum[V], sq[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = sq[e] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S)
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] += get<T, V>(buf[k], e);
    if (GROUPS)
#pragma unroll
        for (int o = 1; o < V; o <<= 1)
#pragma unroll
            for (int e = 0; e < V; e += 2 * o) sum[e] += sum[e + o];
    const float mine = slot.rows(slot.mine, S, a.log_q);
    const float own = mine > 0.f ? 1.f / (mine * (GROUPS ? (float)D : 1.f)) : 0.f;
#pragma unroll
    for (int e = 0; e < NV; ++e) sum[e] = sum_stride(sum_run(sum[e], run), Q);
#pragma unroll
    for (int k = 0; k < K; ++k) forget(buf[k]);
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = get<T, V>(buf[k], e) - sum[GROUPS ? 0 : e] * own;
                sq[e] = fmaf(d, d, sq[e]);
            }
    if (GROUPS)
#pragma unroll
        for (int o = 1; o < V; o <<= 1)
#pragma unroll
            for (int e = 0; e < V; e += 2 * o) sq[e] += sq[e + o];
#pragma unroll
    for (int e = 0; e < NV; ++e) sq[e] = sum_stride(sum_run(sq[e], run), Q);
    if (threadIdx.x % slot.lanes < a.P)
#pragma unroll
        for (int e = 0; e < NV; ++e) {
            sm[slot.mine * width + at + e] = sum[e];
            sm[(slot.count + slot.mine) * width + at + e] = sq[e];
        }
    __syncthreads();
    float mu[V], rs[V];
    const float count = (float)S * (float)D;
    if (GROUPS) {
        if (!on) return;
        double s = 0.0;
        for (int w = 0; w < slot.count; ++w) s += (double)sm[w * width + at];
        const float m = (float)(s / (double)count);
        float q = 0.f;
        for (int w = 0; w < slot.count; ++w) {
            const float rows = slot.rows(w, S, a.log_q) * (float)D;
            const float d = rows > 0.f ? sm[w * width + at] / rows - m : 0.f;
            q += fmaf(rows * d, d, sm[(slot.count + w) * width + at]);
        }
        const float inv = 1.f / sqrtf(q / count + a.eps);
        if (a.mean != nullptr && r == 0 && p % run == 0) {
            a.mean[n * a.G + c0 / D] = m;
            a.rstd[n * a.G + c0 / D] = inv;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            mu[e] = m;
            rs[e] = inv;
        }
    } else {
        float* gv = sm + 2 * slot.count * width;
        const int groups = (a.CB < a.C - slab * a.CB ? a.CB : a.C - slab * a.CB) / D, items = slot.count * D;
        const int share = lanes_for(items), lane = threadIdx.x & (share - 1);
        for (int g = threadIdx.x / share; g < groups; g += NT / share) {
            double s = 0.0, q = 0.0;
            for (int i = lane; i < items; i += share) s += (double)sm[i / D * width + g * D + i % D];
            for (int o = share >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            const float m = (float)(s / (double)count);
            for (int i = lane; i < items; i += share) {
                const int w = i / D, c = g * D + i % D;
                const float rows = slot.rows(w, S, a.log_q);
                const float d = rows > 0.f ? sm[w * width + c] / rows - m : 0.f;
                q += (double)fmaf(rows * d, d, sm[(slot.count + w) * width + c]);
            }
            for (int o = share >> 1; o > 0; o >>= 1) q += __shfl_xor(q, o, 64);
            if (lane == 0) {
                const float inv = 1.f / sqrtf((float)(q / (double)count) + a.eps);
                gv[g] = m;
                gv[groups + g] = inv;
                if (a.mean != nullptr) {
                    a.mean[n * a.G + slab * a.CB / D + g] = m;
                    a.rstd[n * a.G + slab * a.CB / D + g] = inv;
                }
            }
        }
        __syncthreads();
        if (!on) return;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = (p * V + e) / D;
            mu[e] = gv[g];
            rs[e] = gv[groups + g];
        }
    }
    T* y = (T*)a.out + base;
#pragma unroll
    for (int k = 0; k < K; ++k) forget(buf[k]);
    with_act(a.act, [&](auto act) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (r + k * rpb < S) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e)
                    o[e] = act_value(norm_z(norm_xhat(get<T, V>(buf[k], e), mu[e], rs[e]), ga[e], be[e]), decltype(act)::value, a.alpha);
                store_piece<FAR != 0>(piece_at<Q_>(y, at0 + k * step), put<T, V>(o));
            }
    });
}

// LDS: [2][slots][channels of a slab], then with GROUPS [2][slots][groups], without [2][channels] and [2][groups].
template <typename T, int V, int K, int NT, bool GROUPS, int FAR>
__global__ __launch_bounds__(NT) void gn_bwd_held_k(GnArgs a) {
    extern __shared__ float sm[];
    int64_t n;
    int slab;
    if (!unit_of(a, n, slab)) return;
    const int Q = 1 << a.log_q, rpb = NT >> a.log_q, S = (int)a.S, CB = a.CB;
    const int p = threadIdx.x & (Q - 1), r = threadIdx.x >> a.log_q;
    const int c0 = slab * CB + p * V, D = a.D;
    const bool on = p < a.P && c0 < a.C;
    const int64_t base = n * a.S * a.C + slab * CB;
    const uint32_t at0 = (uint32_t)(r * a.C + p * V) * sizeof(T), step = (uint32_t)(rpb * a.C) * sizeof(T);
    typedef Piece<T, V> Q_;
    const T *x = (const T*)a.x + base, *dy = (const T*)a.dy + base;
    Q_ bx[K], bg[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && r + k * rpb < S) {
            bx[k] = load_piece<FAR == 2>(piece_at<const Q_>(x, at0 + k * step));
            bg[k] = load_piece<FAR == 2>(piece_at<const Q_>(dy, at0 + k * step));
        }
    float mu[V], rs[V], ga[V], be[V], s0[V], s1[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        ga[e] = on ? a.gamma[c0 + e] : 0.f;
        be[e] = on ? a.beta[c0 + e] : 0.f;
        if (GROUPS && e > 0) {
            mu[e] = mu[0];
            rs[e] = rs[0];
        } else {
            const int64_t g = n * a.G + (c0 + e) / D;
            mu[e] = on ? a.mean[g] : 0.f;
            rs[e] = on ? a.rstd[g] : 0.f;
        }
        s0[e] = s1[e] = 0.f;
    }
    with_act(a.act, [&](auto act) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (on && r + k * rpb < S) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = norm_xhat(get<T, V>(bx[k], e), mu[e], rs[e]);
                    const float dz = get<T, V>(bg[k], e) * act_slope(norm_z(xh, ga[e], be[e]), decltype(act)::value, a.alpha);
                    s0[e] += dz;
                    s1[e] = fmaf(dz, xh, s1[e]);
                }
            }
#pragma unroll
        for (int e = 0; e < V; ++e) keep_nan(s0[e], s1[e], ga[e], be[e], decltype(act)::value);
    });
#pragma unroll
    for (int k = 0; k < K; ++k) {
        forget(bx[k]);
        forget(bg[k]);
    }
    const Slots<NT> slot(a.log_q);
    const bool writes = threadIdx.x % slot.lanes < a.P;
    float* gs = sm + 2 * slot.count * CB;
    const int run = D / V, groups_cb = CB / D;  // (GROUPS)
    if (GROUPS) {  // the groups' sums of gz, gz xhat
        float g0 = 0.f, g1 = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            g0 = fmaf(s0[e], ga[e], g0);
            g1 = fmaf(s1[e], ga[e], g1);
        }
        g0 = sum_stride(sum_run(g0, run), Q);
        g1 = sum_stride(sum_run(g1, run), Q);
        if (writes) {
            gs[slot.mine * groups_cb + p / run] = g0;
            gs[(slot.count + slot.mine) * groups_cb + p / run] = g1;
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float u = sum_stride(s0[e], Q), w = sum_stride(s1[e], Q);
        if (writes) {
            sm[slot.mine * CB + p * V + e] = u;
            sm[(slot.count + slot.mine) * CB + p * V + e] = w;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * CB; i += NT) {
        const int q = i >= CB, c = i - q * CB;
        double s = 0.0;
        for (int w = 0; w < slot.count; ++w) s += (double)sm[(q * slot.count + w) * CB + c];
        if (slab * CB + c < a.C) a.part[(n * 2 + q) * a.C + slab * CB + c] = (float)s;
        if (!GROUPS) gs[i] = (float)s;
    }
    // dx = rstd gamma dz - rstd mean(gz) - rstd mean(gz xhat) xhat
    float k0[V], k1[V];
    const float inv = 1.f / ((float)S * (float)D);
    if (GROUPS) {
        if (!on) return;
        double u = 0.0, w = 0.0;
        for (int i = 0; i < slot.count; ++i) {
            u += (double)gs[i * groups_cb + p / run];
            w += (double)gs[(slot.count + i) * groups_cb + p / run];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            k0[e] = -rs[0] * ((float)u * inv);
            k1[e] = -rs[0] * ((float)w * inv);
        }
    } else {
        __syncthreads();
        float* gv = gs + 2 * CB;
        const int groups = (CB < a.C - slab * CB ? CB : a.C - slab * CB) / D;
        const int share = lanes_for(D), lane = threadIdx.x & (share - 1);
        for (int g = threadIdx.x / share; g < groups; g += NT / share) {
            double u = 0.0, w = 0.0;
            for (int d = lane; d < D; d += share) {
                const double gamma = (double)a.gamma[slab * CB + g * D + d];
                u += gamma * (double)gs[g * D + d];
                w += gamma * (double)gs[CB + g * D + d];
            }
            for (int o = share >> 1; o > 0; o >>= 1) {
                u += __shfl_xor(u, o, 64);
                w += __shfl_xor(w, o, 64);
            }
            if (lane == 0) {
                gv[g] = (float)u * inv;
                gv[groups + g] = (float)w * inv;
            }
        }
        __syncthreads();
        if (!on) return;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = (p * V + e) / D;
            k0[e] = -rs[e] * gv[g];
            k1[e] = -rs[e] * gv[groups + g];
        }
    }
    T* dx = (T*)a.out + base;
    with_act(a.act, [&](auto act) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (r + k * rpb < S) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    // again, from the pieces: xhat and dz kept from the sums would take twice the registers
                    const float xh = norm_xhat(get<T, V>(bx[k], e), mu[e], rs[e]);
                    const float dz = get<T, V>(bg[k], e) * act_slope(norm_z(xh, ga[e], be[e]), decltype(act)::value, a.alpha);
                    o[e] = fmaf(dz, rs[e] * ga[e], fmaf(xh, k1[e], k0[e]));
                }
                store_piece<FAR != 0>(piece_at<Q_>(dx, at0 + k * step), put<T, V>(o));
            }
    });
}

// ------------------------------------------------------------------------------------------------ streamed
// Workgroup -> (sample, chunk of rows, slab of channels); 256 threads, P = CB / V <= 256 pieces a row, rows r, r + 256 / P, ...
constexpr int kStreamThreads = 256;
__host__ __device__ __forceinline__ bool lanes_share(int P) { return P <= 64 && (P & (P - 1)) == 0; }
// Per chunk and channel.  Forward: mean and sum of squared deviations from it.  A thread sums about the mean of the first U rows it
// takes, which an outlier among them moves by a U-th only; its mean and squares are then joined with the other ones' by counts, across
// lanes, waves and chunks.  So a sum of squares is cut down by L / U of itself at most, L the thread's rows.  (About the chunk's
// first row, should that be the outlier - a border, padding -, it is cut down by as much as the chunk has rows: 0.3 everywhere behind a
// first row of 1e4, 30 M rows, left rstd off by 1.3 %.)  Backward: sum dz, sum dz xhat.
// Eight workgroups a CU: 2048 of them are resident at once (with eight bf16 channels a thread, backward, half of them).
template <typename T, int V, bool BWD>
__global__ __launch_bounds__(kStreamThreads, BWD && V == 8 ? 4 : 8) void gn_sums_k(GnArgs a) {
    extern __shared__ float sm[];  // [2][parts: rows at a time, or waves][channels of a slab] | [3][channels] | [parts]
    constexpr int NT = kStreamThreads, U = BWD ? 2 : V == 8 ? 4 : 8;  // pieces of each tensor in flight
    const int slab = (int)(blockIdx.x % a.slabs);
    const int64_t i = blockIdx.x / a.slabs, n = i / a.chunks, chunk = i % a.chunks;
    const int CB = a.CB, P = a.P, rpb = NT / P;
    const int p = threadIdx.x % P, r = threadIdx.x / P, c0 = slab * CB + p * V;
    const bool on = r < rpb && c0 < a.C;
    const int64_t r0 = chunk * a.rows;
    const int rows = (int)(r0 + a.rows < a.S ? a.rows : a.S - r0);
    // a chunk's base for all threads, 32-bit offsets in it (plan_streamed)
    const int64_t base = (n * a.S + r0) * a.C + slab * CB;
    const uint32_t col = (uint32_t)(p * V) * sizeof(T), pitch = (uint32_t)a.C * sizeof(T);
    typedef const Piece<T, V> Q_;
    const T *x = (const T*)a.x + base, *dy = (const T*)a.dy + base;
    float acc[2][V], mu[V], rs[V], ga[V], be[V];
    Piece<T, V> pivot;  // (forward) the chunk's first row: what means are distances from until the end
    float seen = 0.f;   // (forward) rows in acc
#pragma unroll
    for (int e = 0; e < V; ++e) acc[0][e] = acc[1][e] = 0.f;
    if (on) {
        if (BWD) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int64_t g = n * a.G + (c0 + e) / a.D;
                mu[e] = a.mean[g];
                rs[e] = a.rstd[g];
                ga[e] = a.gamma[c0 + e];
                be[e] = a.beta[c0 + e];
            }
        } else {
            pivot = piece_at<Q_>(x, col);
        }
        const auto row = [&](const Piece<T, V>& bx, const Piece<T, V>& bg, auto act) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (BWD) {
                    const float xh = norm_xhat(get<T, V>(bx, e), mu[e], rs[e]);
                    const float dz = get<T, V>(bg, e) * act_slope(norm_z(xh, ga[e], be[e]), decltype(act)::value, a.alpha);
                    acc[0][e] += dz;
                    acc[1][e] = fmaf(dz, xh, acc[1][e]);
                } else {
                    const float d = get<T, V>(bx, e) - mu[e];
                    acc[0][e] += d;
                    acc[1][e] = fmaf(d, d, acc[1][e]);
                }
            }
        };
        // U rows of this thread, or what is left of them, with all loads ahead of all sums
        const auto block = [&](int at, auto whole, auto act) {
            const auto there = [&](int u) { return decltype(whole)::value || at + u * rpb < rows; };
            Piece<T, V> bx[U], bg[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (there(u)) {
                    bx[u] = piece_at<Q_>(x, col + (at + u * rpb) * pitch);
                    if (BWD) bg[u] = piece_at<Q_>(dy, col + (at + u * rpb) * pitch);
                }
            if constexpr (!BWD) {
                float count = (float)U;
                if (!decltype(whole)::value) {
                    count = 0.f;
#pragma unroll
                    for (int u = 0; u < U; ++u) count += there(u) ? 1.f : 0.f;
                }
                if (seen == 0.f) {  // the first ones
                    const float inv = decltype(whole)::value ? 1.f / (float)U : __builtin_amdgcn_rcpf(count);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float sum = 0.f;
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (there(u)) sum += get<T, V>(bx[u], e);
                        mu[e] = sum * inv;
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) forget(bx[u]);
                }
                seen += count;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (there(u)) row(bx[u], bg[u], act);
        };
        const auto all = [&](auto act) {
            int at = r;
            for (; at + (U - 1) * rpb < rows; at += U * rpb) block(at, std::true_type{}, act);
            if (at < rows) block(at, std::false_type{}, act);
            if (BWD)
#pragma unroll
                for (int e = 0; e < V; ++e) keep_nan(acc[0][e], acc[1][e], ga[e], be[e], decltype(act)::value);
        };
        if (BWD) with_act(a.act, all);
        else all(std::integral_constant<int, SV_ACT_NONE>{});
    }
    if (!BWD && on) {  // sums about mu -> mean and squares about it
        const float inv = seen > 0.f ? __builtin_amdgcn_rcpf(seen) : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float m = acc[0][e] * inv, first = get<T, V>(pivot, e);
            acc[1][e] = fmaf(-acc[0][e], m, acc[1][e]);
            acc[0][e] = seen > 0.f ? mu[e] - first + m : 0.f;
            mu[e] = first;
        }
    }
    // rows together: across lanes where a wave holds whole rows (P a power of two), the rest through LDS
    const bool lanes = lanes_share(P);
    const int held = lanes ? NT / 64 : rpb, mine = lanes ? threadIdx.x >> 6 : r;
    float *s1 = sm + held * CB, *first = s1 + held * CB, *count = first + 3 * CB;
    if (lanes && BWD) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[q][e] = sum_stride(acc[q][e], P);
    } else if (lanes) {
        const float all = sum_stride(seen, P), inv = all > 0.f ? __builtin_amdgcn_rcpf(all) : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float m = sum_stride(seen * acc[0][e], P) * inv, d = acc[0][e] - m;
            acc[1][e] = sum_stride(fmaf(seen * d, d, acc[1][e]), P);
            acc[0][e] = m;
        }
        seen = all;
    }
    if (!BWD && p == 0 && r < rpb && (!lanes || (threadIdx.x & 63) == 0)) count[mine] = seen;
    if (on && (!lanes || (threadIdx.x & 63) < P))
#pragma unroll
        for (int e = 0; e < V; ++e) {
            sm[mine * CB + p * V + e] = acc[0][e];
            s1[mine * CB + p * V + e] = acc[1][e];
            if (!BWD && r == 0) first[p * V + e] = mu[e];
        }
    __syncthreads();
    float* part = a.part + i * 2 * a.C + slab * CB;
    // few channels, many parts (forward): neighbouring lanes share a channel's parts, eight each (2 samples of 500x500x6 f32, whose three
    // pieces a row leave 85 parts, 17.3 -> 15.3 us)
    int shared = 1;
    while (!BWD && shared < 8 && 2 * shared * CB <= NT && 16 * shared <= held) shared <<= 1;
    const int sub = threadIdx.x & (shared - 1);
    for (int c = threadIdx.x / shared; c < CB && slab * CB + c < a.C; c += NT / shared) {
        double u = 0.0, w = 0.0;
        if (BWD) {
            for (int k = 0; k < held; ++k) {
                u += (double)sm[k * CB + c];
                w += (double)s1[k * CB + c];
            }
        } else {  // parts' means and squares -> the chunk's: u = sum n mean, w = sum n mean^2 + squares
            for (int k = sub; k < held; k += shared) {
                const double x = (double)sm[k * CB + c], n0 = (double)count[k] * x;
                u += n0;
                w += fma(n0, x, (double)s1[k * CB + c]);
            }
            for (int o = shared >> 1; o > 0; o >>= 1) {
                u += __shfl_xor(u, o, 64);
                w += __shfl_xor(w, o, 64);
            }
            double inv = (double)__builtin_amdgcn_rcpf((float)rows);
            inv = inv * fma(-(double)rows, inv, 2.0);  // 1 / rows to 2^-44
            const double m = u * inv;
            w = fma(-u, m, w);
            w = w < 0.0 ? 0.0 : w;
            u = (double)first[c] + m;
        }
        const float s = (float)u, q = (float)w;
        if (sub != 0) continue;
        if (BWD || a.groups == nullptr) {
            part[c] = s;
            part[a.C + c] = q;
        }
        if (a.groups != nullptr) {
            first[CB + c] = s;
            first[2 * CB + c] = q;
        }
    }
    if (a.groups == nullptr) return;
    // one slab: the groups' values of this chunk
    __syncthreads();
    const float *chs = first + CB, *chq = first + 2 * CB;
    const int share = lanes_for(a.D), lane = threadIdx.x & (share - 1);
    for (int g = threadIdx.x / share; g < a.G; g += NT / share) {
        double s = 0.0, q = 0.0;
        const double piv = BWD ? 0.0 : (double)chs[g * a.D];
        for (int c = g * a.D + lane; c < (g + 1) * a.D; c += share) {
            if (BWD) {
                s += (double)a.gamma[c] * (double)chs[c];
                q += (double)a.gamma[c] * (double)chq[c];
            } else {
                const double d = (double)chs[c] - piv;
                s += d;
                q += (double)chq[c] + (double)rows * d * d;
            }
        }
        for (int o = share >> 1; o > 0; o >>= 1) {
            s += __shfl_xor(s, o, 64);
            q += __shfl_xor(q, o, 64);
        }
        if (lane == 0) {
            if (!BWD) {
                q -= (double)rows / (double)a.D * s * s;
                s = piv + s / (double)a.D;
            }
            a.groups[(i * 2 + 0) * a.G + g] = (float)s;
            a.groups[(i * 2 + 1) * a.G + g] = !BWD && q < 0.0 ? 0.f : (float)q;
        }
    }
}

// Threads are 16 channels x NT / 16 rows; s, q are a thread's sums over its rows.  Afterwards the first 16 threads hold the sums over
// all rows, in a fixed order.  red: [2][NT / 16][16].
template <int NT>
__device__ __forceinline__ void join16(double& s, double& q, double* red) {
    constexpr int R = NT / 16;
    const int lane = threadIdx.x & 15, w = threadIdx.x >> 4;
    red[w * 16 + lane] = s;
    red[(R + w) * 16 + lane] = q;
    __syncthreads();
    if (w < 8)
        for (int k = w + 8; k < R; k += 8) {
            s += red[k * 16 + lane];
            q += red[(R + k) * 16 + lane];
        }
    // 8 partial sums a channel in the first two waves, 4 rows of 16 lanes in each
    s += __shfl_xor(s, 16, 64);
    q += __shfl_xor(q, 16, 64);
    s += __shfl_xor(s, 32, 64);
    q += __shfl_xor(q, 32, 64);
    if (w == 4) {
        red[lane] = s;
        red[R * 16 + lane] = q;
    }
    __syncthreads();
    if (w == 0) {
        s += red[lane];
        q += red[R * 16 + lane];
    }
}

// The chunks of a sample together, 16 channels a workgroup, 64 chunks at a time: folded[n][2][C] = the sample's mean and sum of
// squared deviations (forward) or sums (backward) per channel.
template <bool BWD>
__global__ __launch_bounds__(1024) void gn_fold_k(GnArgs a) {
    __shared__ double red[2 * 64 * 16];
    const int64_t n = blockIdx.x;
    const int c = blockIdx.y * 16 + (threadIdx.x & 15);
    const float* part = a.part + n * a.chunks * 2 * a.C + c;
    const double piv = !BWD && c < a.C ? (double)part[0] : 0.0;
    double s = 0.0, q = 0.0;
    if (c < a.C) {
#pragma unroll 8
        for (int k = threadIdx.x >> 4; k < a.chunks; k += 64) {
            const double u = (double)part[(int64_t)k * 2 * a.C], v = (double)part[(int64_t)k * 2 * a.C + a.C];
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
    join16<1024>(s, q, red);
    if (threadIdx.x >= 16 || c >= a.C) return;
    if (!BWD) {
        const double m = s / (double)a.S, m2 = q - s * m;
        s = piv + m;
        q = m2 < 0.0 ? 0.0 : m2;
    }
    a.folded[n * 2 * a.C + c] = (float)s;
    a.folded[n * 2 * a.C + a.C + c] = (float)q;
}

// dgamma[c] (+)= sum over parts of part[.][1][c], dbeta[c] (+)= part[.][0][c], for 16 channels.
template <int NT>
__device__ __forceinline__ void fold_params(const float* __restrict__ part, int64_t parts, int C, int c, float* dgamma,
                                            float* dbeta, int accumulate, double* red) {
    double s = 0.0, q = 0.0;
    if (c < C) {
        constexpr int R = NT / 16;
        int64_t i = threadIdx.x >> 4;
        for (; i + 7 * R < parts; i += 8 * R) {
            float x[8], y[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                x[u] = part[(i + u * R) * 2 * C + c];
                y[u] = part[(i + u * R) * 2 * C + C + c];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                s += (double)x[u];
                q += (double)y[u];
            }
        }
        for (; i < parts; i += R) {
            s += (double)part[i * 2 * C + c];
            q += (double)part[i * 2 * C + C + c];
        }
    }
    join16<NT>(s, q, red);
    if (threadIdx.x >= 16 || c >= C) return;
    dgamma[c] = (accumulate ? dgamma[c] : 0.f) + (float)q;
    dbeta[c] = (accumulate ? dbeta[c] : 0.f) + (float)s;
}
__global__ __launch_bounds__(1024) void gn_param_fold_k(const float* __restrict__ part, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta, int64_t parts, int C, int accumulate) {
    __shared__ double red[2 * 64 * 16];
    fold_params<1024>(part, parts, C, blockIdx.x * 16 + (threadIdx.x & 15), dgamma, dbeta, accumulate, red);
}

// The two values of group g of sample n from its D channels' joined ones (a.folded) or from its chunks' ones (a.groups), summed by
// `lanes` neighbouring lanes.  Forward: mean, rstd.  Backward: mean_g(gz), mean_g(gz xhat).
template <bool BWD>
__device__ __forceinline__ void group_values(const GnArgs& a, int64_t n, int g, int lane, int lanes, float& u, float& v) {
    const bool whole = a.groups != nullptr;
    const int terms = whole ? a.chunks : a.D, pitch = whole ? a.G : a.C;  // a term's two values are `pitch` apart
    const int64_t step = whole ? 2 * a.G : 1;                             // two terms
    const float* f = whole ? a.groups + n * a.chunks * 2 * a.G + g : a.folded + n * 2 * a.C + g * a.D;
    const double piv = BWD ? 0.0 : (double)f[0];
    double s = 0.0, q = 0.0;
#pragma unroll 4
    for (int i = lane; i < terms; i += lanes) {
        const double x = (double)f[i * step], y = (double)f[i * step + pitch];
        if (BWD) {
            const double w = whole ? 1.0 : (double)a.gamma[g * a.D + i];
            s += w * x;
            q += w * y;
        } else {  // means and squares about them, of r values each
            const double r = whole ? (double)a.D * (double)((i + 1) * a.rows < a.S ? a.rows : a.S - i * a.rows) : (double)a.S;
            s += r * (x - piv);
            q += y + r * (x - piv) * (x - piv);
        }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        q += __shfl_xor(q, o, 64);
    }
    const double count = (double)a.S * (double)a.D;
    if (BWD) {
        u = (float)(s / count);
        v = (float)(q / count);
    } else {
        const double m = s / count, m2 = q - s * m;
        u = (float)(piv + m);
        v = 1.f / sqrtf((float)((m2 < 0.0 ? 0.0 : m2) / count) + a.eps);
    }
}

template <typename T, int V, bool BWD>
__global__ __launch_bounds__(kStreamThreads, BWD && V == 8 ? 4 : 8) void gn_apply_k(GnArgs a) {
    extern __shared__ float gv[];  // [2][groups that the slab touches]
    constexpr int NT = kStreamThreads, U = BWD || V == 8 ? 2 : 4;
    const int extra = BWD ? (a.C + 15) / 16 : 0;
    if (BWD && (int)blockIdx.x < extra) {  // the first workgroups: dgamma, dbeta
        __shared__ double red[2 * (NT / 16) * 16];
        const bool joined = a.groups == nullptr;
        fold_params<NT>(joined ? a.folded : a.part, joined ? a.N : a.N * a.chunks, a.C, blockIdx.x * 16 + (threadIdx.x & 15),
                        a.dgamma, a.dbeta, a.accumulate, red);
        return;
    }
    // last chunk first: what the statistics pass read last is what the caches still hold
    const int64_t bid = (int64_t)gridDim.x - 1 - blockIdx.x;
    const int slab = (int)(bid % a.slabs);
    const int64_t i = bid / a.slabs, n = i / a.chunks, chunk = i % a.chunks;
    const int first = slab * a.CB, P = a.P, rpb = NT / P;
    const int last = first + a.CB < a.C ? first + a.CB : a.C;
    const int g0 = first / a.D, g1 = (last - 1) / a.D + 1, gs = g1 - g0;
    int lanes = lanes_for(a.groups != nullptr ? a.chunks : a.D);
    while (lanes > 1 && lanes * gs > NT) lanes >>= 1;  // all groups at once: a round of them costs about 1 us
    for (int g = g0 + threadIdx.x / lanes; g < g1; g += NT / lanes) {
        float u, v;
        group_values<BWD>(a, n, g, threadIdx.x % lanes, lanes, u, v);
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
    const int p = threadIdx.x % P, r = threadIdx.x / P, c0 = first + p * V;
    if (r >= rpb || c0 >= a.C) return;
    const int64_t r0 = chunk * a.rows;
    const int rows = (int)(r0 + a.rows < a.S ? a.rows : a.S - r0);
    const int64_t base = (n * a.S + r0) * a.C + first;
    const uint32_t col = (uint32_t)(p * V) * sizeof(T), pitch = (uint32_t)a.C * sizeof(T);
    typedef const Piece<T, V> Q_;
    const T *x = (const T*)a.x + base, *dy = (const T*)a.dy + base;
    T* out = (T*)a.out + base;
    float mu[V], rs[V], ga[V], be[V], k0[V], k1[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = (c0 + e) / a.D;
        ga[e] = a.gamma[c0 + e];
        be[e] = a.beta[c0 + e];
        mu[e] = BWD ? a.mean[n * a.G + g] : gv[g - g0];
        rs[e] = BWD ? a.rstd[n * a.G + g] : gv[gs + g - g0];
        k0[e] = BWD ? -rs[e] * gv[g - g0] : 0.f;  // dx = rstd gamma dz - rstd mean(gz) - rstd mean(gz xhat) xhat
        k1[e] = BWD ? -rs[e] * gv[gs + g - g0] : 0.f;
    }
    with_act(a.act, [&](auto act) {
        const auto row = [&](const Piece<T, V>& bx, const Piece<T, V>& bg, int at) {
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = norm_xhat(get<T, V>(bx, e), mu[e], rs[e]), z = norm_z(xh, ga[e], be[e]);
                if (BWD) {
                    const float dz = get<T, V>(bg, e) * act_slope(z, decltype(act)::value, a.alpha);
                    v[e] = fmaf(dz, rs[e] * ga[e], fmaf(xh, k1[e], k0[e]));
                } else {
                    v[e] = act_value(z, decltype(act)::value, a.alpha);
                }
            }
            // nontemporal: the results then leave the caches' room to what is still to be read again (2 images of 512x512x128 bf16
            // forward 96 -> 85 us, f32 backward 255 -> 236; no size gets slower)
            __builtin_nontemporal_store(put<T, V>(v), &piece_at<Piece<T, V>>(out, col + at * pitch));
        };
        int at = r;
        for (; at + (U - 1) * rpb < rows; at += U * rpb) {
            Piece<T, V> bx[U], bg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                bx[u] = piece_at<Q_>(x, col + (at + u * rpb) * pitch);
                if (BWD) bg[u] = piece_at<Q_>(dy, col + (at + u * rpb) * pitch);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) row(bx[u], bg[u], at + u * rpb);
        }
        for (; at < rows; at += rpb) {
            const Piece<T, V> bx = piece_at<Q_>(x, col + at * pitch);
            row(bx, BWD ? piece_at<Q_>(dy, col + at * pitch) : bx, at);
        }
    });
}

// ------------------------------------------------------------------------------------------------ choice of form
struct GnPlan {
    int V, K, NT, CB, P, slabs;  // K = 0: streamed
    int log_q, far;
    bool groups;
    int64_t rows;
    int chunks;
};

int log2_of(int x) {
    int l = 0;
    while (1 << l < x) ++l;
    return 1 << l == x ? l : -1;
}
int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Largest piece (at most 16 bytes) that divides a row and that every pointer is aligned to.
int piece_of(int C, int size, uintptr_t bits) {
    int v = 16 / size;
    while (v > 1 && (C % v != 0 || bits % ((uintptr_t)v * size) != 0)) v >>= 1;
    return v;
}

// Chunks of the streamed form: `deep` rows a thread, and at most 2048 workgroups, what the chip holds at once; 512 of them, two a CU,
// come first, down to two rows a thread.
void plan_streamed(GnPlan& q, int64_t N, int64_t S, int C, int deep) {
    const int P = C / q.V < kStreamThreads ? C / q.V : kStreamThreads;
    q.K = 0;
    q.NT = kStreamThreads;
    q.P = P;
    q.CB = P * q.V;
    q.slabs = (int)ceil_div(C, q.CB);
    const auto lesser = [](int64_t x, int64_t y) { return x < y ? x : y; };
    const int64_t parts = N * q.slabs, rows = ceil_div(S, kStreamThreads / P);  // rows of one thread
    const int64_t few = lesser(ceil_div(rows, 2), ceil_div(512, parts)), many = lesser(ceil_div(rows, deep), ceil_div(2048, parts));
    const int64_t chunks = few < many ? many : few;
    q.rows = ceil_div(S, chunks);
    const int64_t fit = 0xffffffffll / (4 * (int64_t)C);  // a chunk's offsets have 32 bits
    if (q.rows > fit) q.rows = fit;
    q.chunks = (int)ceil_div(S, q.rows);
}

// The one form whose registers do not suffice (eight bf16 channels of two tensors, channel sums, 1024 threads) is left out.
constexpr bool held_compiled(bool bwd, int size, int piece, int K, int NT, bool groups) {
    return !(bwd && size == 2 && piece == 16 && K == 8 && NT == 1024 && !groups);
}

// Held where a slab of whole groups fits the registers of a workgroup, in the first form of the list that does.
GnPlan gn_plan(int64_t N, int64_t S, int C, int G, int size, uintptr_t bits, bool bwd) {
    // Bytes of a slab's row, pieces a thread, threads.  Rows of a cache line (128 bytes) first, in workgroups of 256 and 512, several
    // a CU, whose phases overlap (1024 samples of 20x20x64 f32 with 512 threads forward 43 us and backward 64; with two
    // workgroups of 1024 threads a CU forward 57, in 64-byte rows backward 78).  A sample of more rows in 64-byte rows with 512
    // threads before 128-byte ones with 1024, of which a CU holds one (512 samples of 32x32x64 bf16 forward 32 against 41 us, 1024 of
    // 30x30x96 94 against 133; backward 59 against 57, 139 against 183) - but for the f32 forward pass of whole groups, of which it
    // holds two (1024 samples of 32x32x64 111 against 125 us).  Below 64 bytes a row the streamed form is faster, and where few
    // workgroups would hold much each: it spreads them.  Fewer than 112 of 8192 pieces and more (37 samples of 31x29x90 bf16, 111
    // workgroups, forward 12.8 against 13.1 us; 50 of 40x40x48, 100 workgroups, 16.4 against 17.5, backward 17.4 against 22.4; 31 of
    // 239x5x64, 62 workgroups, forward the other way, 14.6 against 13.6, backward 14.8 against 18.2), fewer than 48 of 4096 (8 of
    // 32x32x64 f32, 32 workgroups, 9.8 against 11.5 and 9.5 against 11.1; with 100 workgroups, 25 of 32x32x128 bf16, 17.3 against
    // 12.2 and 17.0 against 17.8).
    struct Form {
        int row, K, NT;
        bool two;
    };
    static const Form forms[] = {{128, 2, 256, false}, {128, 4, 256, false}, {128, 8, 256, false}, {128, 8, 512, false}, {128, 8, 1024, true},
                                 {64, 8, 512, false},  {128, 8, 1024, false}, {64, 8, 1024, false},
                                 {128, 16, 1024, false}, {64, 16, 1024, false}};
    GnPlan q{};
    q.V = piece_of(C, size, bits);
    const int D = C / G, unit = D / gcd(D, q.V) * q.V;  // whole groups in whole pieces
    const int piece = q.V * size, most = bwd ? kHeldBwd : kHeldFwd;
    for (const Form& f : forms) {
        int cb = unit;
        if (log2_of(D) >= 0)
            while (cb * 2 * size <= f.row && cb < C) cb *= 2;  // a power of two of pieces, wider than C if that is not one
        else
            cb = f.row / (unit * size) < 1 ? unit : f.row / (unit * size) * unit < C ? f.row / (unit * size) * unit : C;
        const int P = cb / q.V;
        int log_q = 0;
        while (1 << log_q < P) ++log_q;
        const bool groups = log2_of(D) >= 0 && D >= q.V && P == 1 << log_q && P <= 64 && piece >= 8;
        if (cb > kHeldMaxC || 1 << log_q > f.NT || f.K * piece > most || S > (int64_t)f.K * f.NT >> log_q ||
            f.NT / (log_q < 6 ? 64 : 1 << log_q) * cb > kHeldSlots || (f.two && !(groups && size == 4 && !bwd)) ||
            !held_compiled(bwd, size, piece, f.K, f.NT, groups) || N * ceil_div(C, cb) < (f.K * f.NT >= 8192 ? 112 : f.K * f.NT >= 4096 ? 48 : 0))
            continue;
        q.K = f.K;
        q.NT = f.NT;
        q.CB = cb;
        q.P = P;
        q.log_q = log_q;
        q.slabs = (int)ceil_div(C, cb);
        q.groups = groups;
        // Nontemporal stores where a slab's rows are whole sectors of 64 bytes (512 samples of 32x32x64 bf16 forward 41.8 -> 32.2 us,
        // 1024 of 16x16x64 f32 31.2 -> 23.8; with shared sectors 500 samples of 30x31x48 f32 would go from 53 to 91).  Nontemporal
        // loads too where they are whole cache lines and the inputs, of 128 MB and more, hardly come from a cache (1024 of 32x32x64 f32
        // forward 111 -> 104, 16x16x64 backward 50 -> 47; 16x16x64 forward, 67 MB, would go from 24 to 30).
        const auto whole = [&](int unit) { return q.slabs == 1 || (cb * size % unit == 0 && C * size % unit == 0 && bits % unit == 0); };
        const bool large = N * S * C * size * (bwd ? 2 : 1) >= (int64_t)128 << 20;
        q.far = !whole(64) ? 0 : large && whole(128) ? 2 : 1;
        return q;
    }
    // Sixteen rows a thread for two tensors and for narrow pieces, else eight (33 MB of bf16, 64 samples of 90x90x32 with ELU: backward
    // 35.8 us against 37.8, forward 28.2 against 27.3; 100 samples of 30x31x45 bf16 forward 16.4 against 19.8).
    plan_streamed(q, N, S, C, bwd || q.V * size < 8 ? 16 : 8);
    return q;
}

// workspace: [N][2][C] folded sums | [N][chunks][2][C] channels' and [N][chunks][2][G] groups' partial sums, the chunks the most of
// any type and alignment.
int64_t gn_most_chunks(int64_t N, int64_t S, int C) {
    int64_t most = 1;
    for (int v = 1; v <= 8; v *= 2)
        if (C % v == 0) {
            GnPlan q{};
            q.V = v;
            plan_streamed(q, N, S, C, 8);
            if (q.chunks > most) most = q.chunks;
        }
    return most;
}
size_t gn_ws_bytes(int64_t N, int64_t S, int C, int G) {
    return (size_t)N * 2 * (C + (size_t)(C + G) * gn_most_chunks(N, S, C)) * sizeof(float);
}

int gn_check(const char* who, int64_t N, int64_t S, int C, int G, int act, void* ws, size_t ws_bytes) {
    SV_REQUIRE(N >= 0 && S > 0 && C > 0 && C <= kGnMaxC, "%s: bad extents (N=%lld S=%lld C=%d)", who, (long long)N,
               (long long)S, C);
    SV_REQUIRE(G >= 1 && C % G == 0, "%s: %d channels do not split into %d groups", who, C, G);
    SV_REQUIRE(S <= ((int64_t)1 << 40) / C && N <= ((int64_t)1 << 40) / (S * C), "%s: tensor too large", who);
    SV_REQUIRE(act >= SV_ACT_NONE && act <= SV_ACT_SIGMOID, "%s: activation %d unknown", who, act);
    if (N == 0) return SV_OK;
    SV_REQUIRE(N <= (1 << 24) && N * C <= 0x3fffffff, "%s: too many samples", who);
    const size_t need = gn_ws_bytes(N, S, C, G);
    if (ws == nullptr || ws_bytes < need) return fail(SV_E_WORKSPACE, "%s: workspace %zu bytes < required %zu", who, ws_bytes, need);
    return SV_OK;
}

// f(V as an integral constant) for the piece v
template <typename T, typename F>
void with_piece(int v, F f) {
    if constexpr (sizeof(T) == 2)
        if (v == 8) return f(std::integral_constant<int, 8>{});
    if (v == 4) f(std::integral_constant<int, 4>{});
    else if (v == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 1>{});
}

template <typename T, bool BWD, int V, int K, int NT, bool GROUPS, int FAR>
void launch_held_far(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    const dim3 grid((unsigned)held_grid(a.N, q.slabs));
    const size_t slots = NT / (q.log_q < 6 ? 64 : 1 << q.log_q), groups = q.CB / a.D;
    size_t floats;
    if (BWD) floats = 2 * slots * q.CB + (GROUPS ? 2 * slots * groups : 2 * (size_t)q.CB + 2 * groups);
    else floats = GROUPS ? 2 * slots * groups : 2 * slots * q.CB + 2 * groups;
    if constexpr (BWD) hipLaunchKernelGGL((gn_bwd_held_k<T, V, K, NT, GROUPS, FAR>), grid, dim3(NT), floats * sizeof(float), st, a);
    else hipLaunchKernelGGL((gn_fwd_held_k<T, V, K, NT, GROUPS, FAR>), grid, dim3(NT), floats * sizeof(float), st, a);
}

template <typename T, bool BWD, int V, int K, int NT, bool GROUPS>
void launch_held_k(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    if constexpr (GROUPS && V * sizeof(T) == 16) {
        if (q.far == 2) return launch_held_far<T, BWD, V, K, NT, GROUPS, 2>(a, q, st);
        if (q.far == 1) return launch_held_far<T, BWD, V, K, NT, GROUPS, 1>(a, q, st);
    }
    launch_held_far<T, BWD, V, K, NT, GROUPS, 0>(a, q, st);
}

template <typename T, bool BWD, int V, bool GROUPS>
void launch_held_v(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    if (q.NT == 256) {
        if (q.K == 2) launch_held_k<T, BWD, V, 2, 256, GROUPS>(a, q, st);
        else if (q.K == 4) launch_held_k<T, BWD, V, 4, 256, GROUPS>(a, q, st);
        else launch_held_k<T, BWD, V, 8, 256, GROUPS>(a, q, st);
    } else if (q.NT == 512) {
        launch_held_k<T, BWD, V, 8, 512, GROUPS>(a, q, st);
    } else if (q.K == 8) {
        if constexpr (held_compiled(BWD, sizeof(T), V * sizeof(T), 8, 1024, GROUPS)) launch_held_k<T, BWD, V, 8, 1024, GROUPS>(a, q, st);
    } else {
        if constexpr (16 * V * sizeof(T) <= (BWD ? kHeldBwd : kHeldFwd)) launch_held_k<T, BWD, V, 16, 1024, GROUPS>(a, q, st);
    }
}

template <typename T, bool BWD>
void launch_held(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    with_piece<T>(q.V, [&](auto piece) {
        constexpr int V = decltype(piece)::value;
        if constexpr (V * sizeof(T) >= 8) {
            if (q.groups) return launch_held_v<T, BWD, V, true>(a, q, st);
        }
        launch_held_v<T, BWD, V, false>(a, q, st);
    });
}

template <typename T, bool BWD>
void launch_streamed(const GnArgs& a, const GnPlan& q, hipStream_t st) {
    const int64_t main = a.N * q.chunks * q.slabs;
    const int held = lanes_share(q.P) ? kStreamThreads / 64 : kStreamThreads / q.P;
    const size_t lds = ((2 * (size_t)held + 3) * q.CB + held) * sizeof(float);  // at most 41 KB
    const size_t lds_apply = 2 * ((size_t)q.CB / a.D + 2) * sizeof(float);
    with_piece<T>(q.V, [&](auto piece) {
        constexpr int V = decltype(piece)::value;
        hipLaunchKernelGGL((gn_sums_k<T, V, BWD>), dim3((unsigned)main), dim3(kStreamThreads), lds, st, a);
        if (a.groups == nullptr)
            hipLaunchKernelGGL((gn_fold_k<BWD>), dim3((unsigned)a.N, (unsigned)ceil_div(a.C, 16)), dim3(1024), 0, st, a);
        hipLaunchKernelGGL((gn_apply_k<T, V, BWD>), dim3((unsigned)(main + (BWD ? ceil_div(a.C, 16) : 0))),
                           dim3(kStreamThreads), lds_apply, st, a);
    });
}

template <typename T, bool BWD>
int launch(const char* who, GnArgs& a, void* workspace, hipStream_t st) {
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)a.dy;
    const GnPlan q = gn_plan(a.N, a.S, a.C, a.G, sizeof(T), bits, BWD);
    a.CB = q.CB;
    a.P = q.P;
    a.log_q = q.log_q;
    a.slabs = q.slabs;
    a.rows = q.rows;
    a.chunks = q.chunks;
    a.folded = (float*)workspace;
    const int64_t grid = q.K > 0 ? held_grid(a.N, q.slabs) : a.N * q.chunks * q.slabs + ceil_div(a.C, 16);
    const int64_t threads = q.K > 0 ? grid * q.NT : grid * kStreamThreads;  // (gn_fold_k: N * 1024)
    SV_REQUIRE(threads <= 0xffffffffll && (q.K > 0 || a.N < (1 << 22)), "%s: too many samples for one launch", who);
    if (q.K > 0) {
        a.part = (float*)workspace;
        launch_held<T, BWD>(a, q, st);
        if (BWD)
            hipLaunchKernelGGL(gn_param_fold_k, dim3((unsigned)ceil_div(a.C, 16)), dim3(1024), 0, st, a.part, a.dgamma, a.dbeta,
                               a.N, a.C, a.accumulate);
    } else {
        a.part = a.folded + a.N * 2 * a.C;
        // Whole groups in a slab and few chunks: the second pass joins the groups' values itself, which saves a launch (32 samples of
        // 128x128x32 bf16 forward 27.0 -> 25.2 us, backward 38.1 -> 37.1; one of 18x67x10 f32 10.0 -> 8.8).  All of its workgroups read
        // all of a sample's values: more than 10 MB in all cost more than the launch (two samples of 512x512x32 bf16, 1024 chunks
        // each, 28.5 -> 35.3).  Backward, its first workgroups also add the channels' sums of all chunks.
        if (q.slabs == 1 && a.N * q.chunks * q.chunks * a.G <= 5 << 18 && (!BWD || a.N * q.chunks <= 2048))
            a.groups = a.part + a.N * q.chunks * 2 * a.C;
        launch_streamed<T, BWD>(a, q, st);
    }
    return check_launch(who);
}

}  // namespace
}  // namespace sv
