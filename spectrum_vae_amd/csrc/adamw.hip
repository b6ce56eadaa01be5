// AdamW over a list of tensors in one launch, with moments in 32 or in 8 bits, and the gradients' global norm.
//   t = count + 1;  lr = lr0 rate^(count / steps);  alpha = lr sqrt(1 - b2^t) / (1 - b1^t)
//   s = grad_scale, or grad_scale clip / max(clip, grad_scale ||g||)
//   g' = s g;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   theta -= lr decay theta;  theta -= alpha m / (sqrt(v) + eps)
//
// Moments in 8 bits: blocks of 256 elements of one tensor, one exponent byte e a block (255: a value of the block is not finite).
// A first moment is sign, 4 exponent and 3 mantissa bits, a second moment 5 exponent and 3 mantissa bits; a code stands for the
// float whose bits are code << 20, times 2^(e - top), top = 15 or 31.  e is the exponent of the block's largest magnitude once
// its mantissa is rounded up to 3 bits, so rounding up never leaves the code's range.  Powers of two as scales lose nothing: the
// codes are floating-point themselves, and scaling by them is exact.
// The rounding is by random bits (up with a probability equal to the distance to the code below): with b2 = 0.999 a second moment
// changes by 0.1 % a step, and rounding to nearest at 3 bits (steps of 12 %) would never move it.  A positive second moment never
// becomes 0 (the step would divide by eps alone).  All arithmetic is in 32 bits with every rounding spelled out; theta's step
// uses the moments before they are rounded.
//
// What bounds it: the memory.  A weight moves 28 bytes with 32-bit moments (theta, m, v both ways, the gradient), 16.02 with 8-bit
// ones, for about 16 flops.  Measured where a copy runs at 5.3 TB/s and a launch that does next to nothing takes 3.5 us:
//   101 M weights   adamw_k<32>  482 us  5.9 TB/s;  grad_norm_k  68 us  5.9;  adamw_k<8>  304 us  5.3;  adamw_decode_k  94 us  5.4
//   0.8 M weights   adamw_k<8> with a bf16 copy  7.8 us;  adamw_decode_k  2.8 us
//   12 thousand weights in 12 tensors   adamw_k<32>  4.4 us
#include <algorithm>
#include <new>
#include <vector>

#include "common.h"

namespace sv {
namespace {

constexpr int kBlock = 256;        // elements of an 8-bit block
constexpr int kChunk = 4096;       // elements of one tensor that a workgroup updates at a time
constexpr int kNormParts = 2048;   // most workgroups (partial sums) of the norm launch: eight a CU

// A pointer read from memory is not known to point there: without this its accesses would be flat ones, which also go by LDS.
#define SV_GLOBAL __attribute__((address_space(1)))

// One entry of the plan on the device: up to kChunk consecutive elements of one tensor.  Pointers are to the chunk's own first
// element, so a workgroup gets to its data through a single dependent load.
struct Chunk {
    float* theta;
    float* grad;
    void* m;
    void* v;
    uint8_t* m_exp;
    uint8_t* v_exp;
    __bf16* theta_lp;
    int64_t block;  // its first 8-bit block's number among those of all tensors (the position in the random stream)
    int32_t n;
    float decay;
    int32_t vec;    // every pointer takes 4-element accesses
    int32_t pad;
};

constexpr unsigned kTickets = 32;
struct alignas(128) Ticket {
    unsigned count;
};
// device image: Ticket[kTickets + 1] (zero between launches), Chunk[n_chunks]

struct StepArgs {
    Ticket* tickets;
    const Chunk* chunks;
    int64_t n_chunks;
    int64_t* state;
    const double* norm_parts;
    double lr0, log_beta1, log_beta2, log_rate;
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, grad_scale, clip;
    int decay_steps, staircase, zero_grad, n_norm_parts, log_split;
    uint64_t seed;
};

__device__ __forceinline__ float code_value(uint32_t bits, int e, int top) {
    return e == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(__uint_as_float(bits), e - top);
}
__device__ __forceinline__ float first_value(uint32_t code, int e) {
    const float v = code_value((code & 0x7fu) << 20, e, 15);
    return code & 0x80u ? -v : v;
}
__device__ __forceinline__ float second_value(uint32_t code, int e) { return code_value(code << 20, e, 31); }

// Exponent of the block's largest magnitude (given as its bits) with the mantissa rounded up to 3 bits; 255: not finite.
__device__ __forceinline__ int block_exponent(uint32_t largest) {
    const uint32_t e = (largest + 0xfffffu) >> 23;
    return e > 255u ? 255 : (int)e;
}
// The magnitude's code: its bits at the code's scale, with 16 random bits added below the code's last bit, cut off.
__device__ __forceinline__ uint32_t code_of(float x, int e, int top, uint32_t random16) {
    const uint32_t bits = __float_as_uint(ldexpf(x, top - e)) & 0x7fffffffu;
    return (bits + (random16 << 4)) >> 20;
}
__device__ __forceinline__ uint32_t first_code(float m, int e, uint32_t random16) {
    return e == 255 ? 0u : code_of(m, e, 15, random16) | (__float_as_uint(m) >> 31 << 7);
}
__device__ __forceinline__ uint32_t second_code(float v, int e, uint32_t random16) {
    if (e == 255) return 0u;
    const uint32_t c = code_of(v, e, 31, random16);
    return c == 0u && v > 0.f ? 1u : c;
}

// Root and quotient are the hardware's (1 ulp each): they only enter theta's step.
__device__ __forceinline__ void update(float& th, float& m, float& v, float g, const StepArgs& a, float scale, float alpha,
                                       float lr_decay) {
#pragma clang fp contract(off)
    const float gs = g * scale;
    m = a.beta1 * m + a.one_minus_beta1 * gs;
    v = a.beta2 * v + a.one_minus_beta2 * (gs * gs);
    th = th - lr_decay * th;
    th = th - (alpha * m) * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) + a.eps);
}

// Maximum over a wave in every lane, one vector instruction a step (no LDS): within a row of 16 lanes by data-parallel
// primitives, between rows by lane swaps.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
    return w > v ? w : v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0xB1>(v);   // lane ^ 1
    v = dpp_max<0x4E>(v);   // lane ^ 2
    v = dpp_max<0x141>(v);  // the other half of 8
    v = dpp_max<0x140>(v);  // the other half of 16
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = r[0] > r[1] ? r[0] : r[1];
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] > r[1] ? r[0] : r[1];
}

typedef float Float4 __attribute__((ext_vector_type(4)));
typedef uint32_t Word2 __attribute__((ext_vector_type(2)));

// Partial sums of squares of the gradients, one a workgroup, squared and added in f64: a square of any finite float is a number there,
// so one gradient above 1.8e19 (or all of them below 1e-19) leaves a norm to clip by.  The launch stays at the memory's rate with
// four chains a thread (a clipped step of 101 M weights 561 us, with squares in f32 562).  A workgroup's next entry is asked for ahead
// of the current one's data.
__global__ __launch_bounds__(256) void grad_norm_k(const Chunk* __restrict__ chunks, int64_t n_chunks, double* __restrict__ parts) {
    __shared__ double red[4];
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    int64_t k = blockIdx.x;
    const float* g = k < n_chunks ? chunks[k].grad : nullptr;
    int n = k < n_chunks ? chunks[k].n : 0, vec = k < n_chunks ? chunks[k].vec : 0;
    while (k < n_chunks) {
        k += gridDim.x;
        const Chunk* next = chunks + (k < n_chunks ? k : 0);
        const float* g_next = next->grad;
        const int n_next = next->n, vec_next = next->vec;
        if (vec && n == kChunk) {
            Float4 q[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = ((const SV_GLOBAL Float4*)g)[threadIdx.x + 256 * u];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fma((double)q[u][e], (double)q[u][e], sum[e]);
        } else {
            for (int i = threadIdx.x; i < n; i += 256) {
                const double d = (double)((const SV_GLOBAL float*)g)[i];
                sum[0] = fma(d, d, sum[0]);
            }
        }
        g = g_next;
        n = n_next;
        vec = vec_next;
    }
    double all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = all;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// Four consecutive elements of a lane: VEC as one access, else the first `mine` one by one (the others read as 0).
// FAR: around the caches (nontemporal), for data that will not be there any more when it is used again.
template <bool FAR, typename E, typename Q>
__device__ __forceinline__ void load4(const E* generic, bool vec, int mine, E (&out)[4]) {
    const SV_GLOBAL E* p = (const SV_GLOBAL E*)generic;
    if (vec) {
        const Q q = FAR ? __builtin_nontemporal_load((const SV_GLOBAL Q*)p) : *(const SV_GLOBAL Q*)p;
        __builtin_memcpy(out, &q, sizeof(q));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = e < mine ? p[e] : (E)0;
    }
}
template <bool FAR, typename E, typename Q>
__device__ __forceinline__ void store4(E* generic, bool vec, int mine, const E (&in)[4]) {
    SV_GLOBAL E* p = (SV_GLOBAL E*)generic;
    if (vec) {
        Q q;
        __builtin_memcpy(&q, in, sizeof(q));
        if (FAR) __builtin_nontemporal_store(q, (SV_GLOBAL Q*)p);
        else *(SV_GLOBAL Q*)p = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < mine) p[e] = in[e];
    }
}

template <bool FAR>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* generic, bool vec, int mine) {
    const SV_GLOBAL uint8_t* p = (const SV_GLOBAL uint8_t*)generic;
    if (vec) return FAR ? __builtin_nontemporal_load((const SV_GLOBAL uint32_t*)p) : *(const SV_GLOBAL uint32_t*)p;
    uint32_t w = 0;
    for (int e = 0; e < mine; ++e) w |= (uint32_t)p[e] << 8 * e;
    return w;
}
template <bool FAR>
__device__ __forceinline__ void store_codes(uint8_t* generic, bool vec, int mine, uint32_t w) {
    SV_GLOBAL uint8_t* p = (SV_GLOBAL uint8_t*)generic;
    if (vec) {
        if (FAR) __builtin_nontemporal_store(w, (SV_GLOBAL uint32_t*)p);
        else *(SV_GLOBAL uint32_t*)p = w;
    } else {
        for (int e = 0; e < mine; ++e) p[e] = (uint8_t)(w >> 8 * e);
    }
}

// What a lane holds of a block of 256 elements.
template <int BITS, bool FAR>
struct Held {
    float th[4], g[4], m[4], v[4];
    uint32_t mc, vc;  // four codes each
    int me, ve, mine;
    bool vec;

    __device__ __forceinline__ void load(const Chunk& c, int b, int lane) {
        const uint32_t i = b * kBlock + 4 * lane;  // (unsigned: offsets then need no register pair)
        const int left = c.n - (int)i;
        mine = left >= 4 ? 4 : left > 0 ? left : 0;
        vec = c.vec && c.n - b * kBlock >= kBlock;  // the same for the whole wave
        load4<FAR, float, Float4>(c.theta + i, vec, mine, th);
        load4<FAR, float, Float4>(c.grad + i, vec, mine, g);
        if (BITS == 8) {
            me = ((const SV_GLOBAL uint8_t*)c.m_exp)[b];
            ve = ((const SV_GLOBAL uint8_t*)c.v_exp)[b];
            mc = load_codes<FAR>((const uint8_t*)c.m + i, vec, mine);
            vc = load_codes<FAR>((const uint8_t*)c.v + i, vec, mine);
        } else {
            load4<FAR, float, Float4>((const float*)c.m + i, vec, mine, m);
            load4<FAR, float, Float4>((const float*)c.v + i, vec, mine, v);
        }
    }

    __device__ __forceinline__ void step(const Chunk& c, int b, int lane, const StepArgs& a, float scale, float alpha,
                                         float lr_decay, uint64_t key) {
        const uint32_t i = b * kBlock + 4 * lane;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (BITS == 8) {
                m[e] = first_value(mc >> 8 * e & 0xffu, me);
                v[e] = second_value(vc >> 8 * e & 0xffu, ve);
            }
            update(th[e], m[e], v[e], g[e], a, scale, alpha, lr_decay);
        }
        if (BITS == 8) {
            uint32_t ml = 0, vl = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t mb = e < mine ? __float_as_uint(m[e]) & 0x7fffffffu : 0u;
                const uint32_t vb = e < mine ? __float_as_uint(v[e]) & 0x7fffffffu : 0u;
                ml = mb > ml ? mb : ml;
                vl = vb > vl ? vb : vl;
            }
            me = block_exponent(wave_max(ml));
            ve = block_exponent(wave_max(vl));
            const uint64_t pair = (uint64_t)((c.block + b) * (kBlock / 2) + 2 * lane);
            const uint64_t h0 = mix64(pair ^ key), h1 = mix64((pair + 1) ^ key);
            const uint32_t r[4] = {(uint32_t)h0, (uint32_t)(h0 >> 32), (uint32_t)h1, (uint32_t)(h1 >> 32)};
            mc = vc = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mc |= first_code(m[e], me, r[e] & 0xffffu) << 8 * e;
                vc |= second_code(v[e], ve, r[e] >> 16) << 8 * e;
            }
            store_codes<FAR>((uint8_t*)c.m + i, vec, mine, mc);
            store_codes<FAR>((uint8_t*)c.v + i, vec, mine, vc);
            if (lane == 0) {
                ((SV_GLOBAL uint8_t*)c.m_exp)[b] = (uint8_t)me;
                ((SV_GLOBAL uint8_t*)c.v_exp)[b] = (uint8_t)ve;
            }
        } else {
            store4<FAR, float, Float4>((float*)c.m + i, vec, mine, m);
            store4<FAR, float, Float4>((float*)c.v + i, vec, mine, v);
        }
        store4<FAR, float, Float4>(c.theta + i, vec, mine, th);
        if (c.theta_lp != nullptr) {
            const __bf16 lp[4] = {(__bf16)th[0], (__bf16)th[1], (__bf16)th[2], (__bf16)th[3]};
            store4<FAR, __bf16, Word2>(c.theta_lp + i, vec, mine, lp);
        }
        if (a.zero_grad) {
            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
            store4<FAR, float, Float4>(c.grad + i, vec, mine, zero);
        }
    }
};

// The update's common scalars, worked out by every workgroup: {alpha, lr, gradient scale}.  The three powers are one
// call of exp on three lanes (b^t = exp(t log b)).
__device__ __forceinline__ void schedule(const StepArgs& a, int64_t it, double norm2, float* out) {
    const int lane = threadIdx.x & 63;
    double e = 0.0;
    if (a.decay_steps > 0) {
        e = (double)it / (double)a.decay_steps;
        if (a.staircase) e = floor(e);
    }
    const double t = (double)(it + 1);
    const double power = exp(lane == 0 ? t * a.log_beta1 : lane == 1 ? t * a.log_beta2 : e * a.log_rate);
    const double p1 = __shfl(power, 0, 64), p2 = __shfl(power, 1, 64), rate = __shfl(power, 2, 64);
    if (lane != 0) return;
    const double lr = a.lr0 * rate;
    out[0] = (float)(lr * sqrt(1.0 - p2) / (1.0 - p1));  // 1 - b^t loses at most 2^-53 / (1 - b) of itself
    out[1] = (float)lr;
    out[2] = a.grad_scale;
    if (a.n_norm_parts > 0) {
        const double norm = fabs((double)a.grad_scale) * sqrt(norm2);
        // a norm that is not finite leaves nothing finite, as the clip of Keras
        const float clip = norm > a.clip ? (float)((double)a.clip / norm) : 1.f;
        out[2] = norm - norm == 0.0 ? a.grad_scale * clip : __uint_as_float(0x7fc00000u);
    }
}

// Whether this is the last workgroup of the launch to get here (one thread asks).  With more than 64 of them arrivals are counted
// in kTickets places of a cache line each first: on a single counter, 850 workgroups queue for 8 us.  All counters are left
// zero.
__device__ __forceinline__ bool last_of(Ticket& t, unsigned all) {
    if (__hip_atomic_fetch_add(&t.count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != all - 1) return false;
    __hip_atomic_store(&t.count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}
__device__ __forceinline__ bool last_to_arrive(Ticket* t) {
    if (gridDim.x <= 64) return last_of(t[kTickets], gridDim.x);
    const unsigned at = blockIdx.x % kTickets;
    return last_of(t[at], (gridDim.x - at + kTickets - 1) / kTickets) && last_of(t[kTickets], kTickets);
}

// A wave takes blocks of 256 elements, four a lane: every 4 * 2^log_split-th block of a chunk, 2^log_split workgroups a chunk (so
// that few chunks spread over more CUs).  The first block is asked for before the common scalars are worked out.
// A CU holds kResident workgroups (64 registers a thread, 80 with 8-bit moments); no launch has more of them at once.
template <int BITS> constexpr int kResident = BITS == 8 ? 6 : 8;
template <int BITS, bool FAR>
__global__ __launch_bounds__(256, kResident<BITS>) void adamw_k(StepArgs a) {
    __shared__ float s[3];
    __shared__ double red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t it = a.state[0], items = a.n_chunks << a.log_split;
    Held<BITS, FAR> h;
    int64_t k = blockIdx.x;  // item: chunk k >> log_split, its blocks from 4 times the rest on
    int first = 4 * (int)(k & ((1 << a.log_split) - 1)) + wave;
    Chunk c{};
    if (k < items) {
        c = a.chunks[k >> a.log_split];
        if (first * kBlock < c.n) h.load(c, first, lane);
    }
    double norm2 = 0.0;
    if (a.n_norm_parts > 0) {
        for (int i = threadIdx.x; i < a.n_norm_parts; i += 256) norm2 += a.norm_parts[i];
        for (int o = 32; o > 0; o >>= 1) norm2 += __shfl_xor(norm2, o, 64);
        if (lane == 0) red[wave] = norm2;
        __syncthreads();
        norm2 = red[0] + red[1] + red[2] + red[3];
    }
    if (wave == 0) schedule(a, it, norm2, s);
    __syncthreads();
    const float alpha = s[0], lr = s[1], scale = s[2];
    const uint64_t key = mix64(mix64((uint64_t)it) ^ a.seed);
    while (k < items) {
        const float lr_decay = lr * c.decay;
        for (int b = first; b * kBlock < c.n; b += 4 << a.log_split) {
            if (b != first || k != blockIdx.x) h.load(c, b, lane);
            h.step(c, b, lane, a, scale, alpha, lr_decay, key);
        }
        k += gridDim.x;
        if (k < items) {
            first = 4 * (int)(k & ((1 << a.log_split) - 1)) + wave;
            c = a.chunks[k >> a.log_split];
        }
    }
    // the workgroup that arrives last advances the count: every workgroup has read it by then
    __syncthreads();
    if (threadIdx.x == 0 && last_to_arrive(a.tickets)) {
        a.state[0] = it + 1;
        reinterpret_cast<float*>(a.state + 1)[0] = alpha;
        reinterpret_cast<float*>(a.state + 1)[1] = lr;
    }
}

// Four codes a thread where codes and output allow it (VEC), n4 groups of four; then the last n % 4 one by one.
template <bool SECOND, bool FAR>
__global__ __launch_bounds__(256) void adamw_decode_k(const uint8_t* __restrict__ code, const uint8_t* __restrict__ exps,
                                                       float* __restrict__ out, int64_t n, int64_t n4) {
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = (int64_t)gridDim.x * 256;
    for (int64_t i = first; i < n4; i += stride) {
        const uint32_t q = reinterpret_cast<const uint32_t*>(code)[i];
        const int e = exps[i / (kBlock / 4)];
        Float4 o;
        o.x = SECOND ? second_value(q & 0xffu, e) : first_value(q & 0xffu, e);
        o.y = SECOND ? second_value(q >> 8 & 0xffu, e) : first_value(q >> 8 & 0xffu, e);
        o.z = SECOND ? second_value(q >> 16 & 0xffu, e) : first_value(q >> 16 & 0xffu, e);
        o.w = SECOND ? second_value(q >> 24, e) : first_value(q >> 24, e);
        if (FAR) __builtin_nontemporal_store(o, reinterpret_cast<Float4*>(out) + i);
        else reinterpret_cast<Float4*>(out)[i] = o;
    }
    for (int64_t i = 4 * n4 + first; i < n; i += stride)
        out[i] = SECOND ? second_value(code[i], exps[i / kBlock]) : first_value(code[i], exps[i / kBlock]);
}

struct Span {
    uintptr_t begin, end;
    int tensor;
};
// The first two ranges that share a byte, or -1.
int overlap(std::vector<Span>& spans, int* other) {
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i].begin < spans[i - 1].end) {
            *other = spans[i].tensor;
            return spans[i - 1].tensor;
        }
    return -1;
}

int64_t plan_chunks(const sv_adamw_tensor* t, int n_tensors) {
    int64_t chunks = 0;
    for (int i = 0; i < n_tensors; ++i) chunks += ceil_div(t[i].n, kChunk);
    return chunks;
}

int plan_check(const char* who, const sv_adamw_tensor* t, int n_tensors, int state_bits) {
    SV_REQUIRE(t != nullptr && n_tensors >= 1 && n_tensors <= (1 << 20), "%s: 1..%d tensors", who, 1 << 20);
    SV_REQUIRE(state_bits == 8 || state_bits == 32, "%s: moments have 8 or 32 bits, not %d", who, state_bits);
    int64_t total = 0;
    std::vector<Span> spans;
    for (int i = 0; i < n_tensors; ++i) {
        const sv_adamw_tensor& e = t[i];
        SV_REQUIRE(e.n >= 0 && e.n <= ((int64_t)1 << 40), "%s: tensor %d has %lld elements", who, i, (long long)e.n);
        SV_REQUIRE(e.weight_decay >= 0.f && e.weight_decay < 3.4e38f, "%s: tensor %d: weight decay out of range", who, i);
        if (e.n == 0) continue;
        total += e.n;
        SV_REQUIRE(total <= ((int64_t)1 << 40), "%s: too many elements", who);
        SV_REQUIRE(e.theta && e.grad && e.m && e.v, "%s: tensor %d: null buffer", who, i);
        SV_REQUIRE(state_bits == 32 || (e.m_exp && e.v_exp), "%s: tensor %d: 8-bit moments need their exponents", who, i);
        const int64_t blocks = ceil_div(e.n, kBlock), each = state_bits == 8 ? 1 : 4;
        bool ok = true;
        auto add = [&](const void* p, int64_t bytes, uintptr_t align) {
            spans.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, i});
            ok = ok && (uintptr_t)p % align == 0;
        };
        add(e.theta, 4 * e.n, 4);
        add(e.grad, 4 * e.n, 4);
        add(e.m, each * e.n, each);
        add(e.v, each * e.n, each);
        if (state_bits == 8) {
            add(e.m_exp, blocks, 1);
            add(e.v_exp, blocks, 1);
        }
        if (e.theta_bf16) add(e.theta_bf16, 2 * e.n, 2);
        SV_REQUIRE(ok, "%s: tensor %d: a buffer is not aligned to its elements", who, i);
    }
    int other = 0;
    const int one = overlap(spans, &other);
    SV_REQUIRE(one < 0, "%s: buffers of tensors %d and %d overlap", who, one, other);
    return SV_OK;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" {

size_t sv_adamw_plan_bytes(const sv_adamw_tensor* tensors, int n_tensors, int64_t* n_chunks) {
    if (tensors == nullptr || n_chunks == nullptr || n_tensors < 1) return 0;
    for (int i = 0; i < n_tensors; ++i)
        if (tensors[i].n < 0 || tensors[i].n > ((int64_t)1 << 40)) return 0;
    *n_chunks = plan_chunks(tensors, n_tensors);
    return (kTickets + 1) * sizeof(Ticket) + (size_t)*n_chunks * sizeof(Chunk);
}

int sv_adamw_plan_fill(const sv_adamw_tensor* tensors, int n_tensors, int state_bits, void* image, size_t image_bytes) {
    try {
        int rc = plan_check("sv_adamw_plan_fill", tensors, n_tensors, state_bits);
        if (rc) return rc;
        int64_t n_chunks = 0;
        const size_t need = sv_adamw_plan_bytes(tensors, n_tensors, &n_chunks);
        if (image == nullptr || image_bytes < need)
            return fail(SV_E_WORKSPACE, "sv_adamw_plan_fill: image %zu bytes < required %zu", image_bytes, need);
        memset(image, 0, (kTickets + 1) * sizeof(Ticket));
        Chunk* chunk = (Chunk*)((char*)image + (kTickets + 1) * sizeof(Ticket));
        int64_t block = 0;
        for (int i = 0; i < n_tensors; ++i) {
            const sv_adamw_tensor& e = tensors[i];
            const uintptr_t state_align = state_bits == 8 ? 4 : 16;
            const bool vec = (uintptr_t)e.theta % 16 == 0 && (uintptr_t)e.grad % 16 == 0 && (uintptr_t)e.m % state_align == 0 &&
                             (uintptr_t)e.v % state_align == 0 && (uintptr_t)e.theta_bf16 % 8 == 0;
            for (int64_t at = 0; at < e.n; at += kChunk) {
                const int64_t left = e.n - at, each = state_bits == 8 ? 1 : 4, b = at / kBlock;
                *chunk++ = Chunk{e.theta + at, e.grad + at, (char*)e.m + each * at, (char*)e.v + each * at,
                                 state_bits == 8 ? e.m_exp + b : nullptr, state_bits == 8 ? e.v_exp + b : nullptr,
                                 e.theta_bf16 ? (__bf16*)e.theta_bf16 + at : nullptr, block + b,
                                 (int32_t)(left < kChunk ? left : kChunk), e.weight_decay, vec, 0};
            }
            block += ceil_div(e.n, kBlock);
        }
        return SV_OK;
    } catch (const std::bad_alloc&) {
        return fail(SV_E_INVALID, "sv_adamw_plan_fill: out of host memory");
    }
}

size_t sv_adamw_workspace_bytes(void) { return kNormParts * sizeof(double); }

int sv_adamw_step(void* plan, int64_t n_chunks, int state_bits, int64_t* step_state, double lr0,
                  double beta1, double beta2, float eps, int decay_steps, double decay_rate, int staircase, float grad_scale,
                  float clip_norm, uint64_t seed, int zero_grad, void* workspace, size_t workspace_bytes, sv_stream_t stream) {
    SV_REQUIRE(plan != nullptr && step_state != nullptr && n_chunks >= 0, "sv_adamw_step: bad arguments");
    SV_REQUIRE((uintptr_t)plan % 128 == 0 && (uintptr_t)step_state % 8 == 0, "sv_adamw_step: plan must be 128-byte, state 8-byte aligned");
    SV_REQUIRE(state_bits == 8 || state_bits == 32, "sv_adamw_step: moments have 8 or 32 bits, not %d", state_bits);
    SV_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "sv_adamw_step: betas out of range");
    // the step's root takes second moments below 1.2e-38 as 0, which is 1e-19 in it: nothing next to such an epsilon
    SV_REQUIRE(eps >= 1e-12f, "sv_adamw_step: epsilon must be at least 1e-12");
    SV_REQUIRE(clip_norm >= 0.f && (decay_steps <= 0 || decay_rate > 0.0), "sv_adamw_step: the decay rate must be positive, the clip not negative");
    SV_REQUIRE(clip_norm == 0.f || (workspace != nullptr && (uintptr_t)workspace % 8 == 0), "sv_adamw_step: clipping needs a workspace");
    if (clip_norm > 0.f && workspace_bytes < sv_adamw_workspace_bytes())
        return fail(SV_E_WORKSPACE, "sv_adamw_step: workspace %zu bytes < required %zu", workspace_bytes, sv_adamw_workspace_bytes());
    hipStream_t st = to_stream(stream);
    StepArgs a{};
    a.tickets = (Ticket*)plan;
    a.chunks = (const Chunk*)(a.tickets + kTickets + 1);
    a.n_chunks = n_chunks;
    a.state = step_state;
    a.lr0 = lr0;
    a.log_beta1 = log(beta1);
    a.log_beta2 = log(beta2);
    a.log_rate = decay_steps > 0 ? log(decay_rate) : 0.0;
    a.beta1 = (float)beta1;
    a.beta2 = (float)beta2;
    a.one_minus_beta1 = (float)(1.0 - beta1);
    a.one_minus_beta2 = (float)(1.0 - beta2);
    a.eps = eps;
    a.grad_scale = grad_scale;
    a.clip = clip_norm;
    a.decay_steps = decay_steps;
    a.staircase = staircase;
    a.zero_grad = zero_grad;
    a.seed = seed;
    if (clip_norm > 0.f && n_chunks > 0) {
        a.norm_parts = (const double*)workspace;
        a.n_norm_parts = (int)(n_chunks < kNormParts ? n_chunks : kNormParts);
        hipLaunchKernelGGL(grad_norm_k, dim3(a.n_norm_parts), dim3(256), 0, st, a.chunks, n_chunks, (double*)workspace);
    }
    const int most = 256 * (state_bits == 8 ? kResident<8> : kResident<32>);
    a.log_split = 4 * n_chunks <= most ? 2 : 2 * n_chunks <= most ? 1 : 0;  // a block a wave where the chip holds that at once
    const int64_t items = n_chunks << a.log_split;
    const int grid = (int)(items < 1 ? 1 : items < most ? items : most);
    // more than the caches between the chip and the memory hold (256 MB): nothing of it is found there at the next step
    // (101 M weights: 555 against 515 us with 32-bit moments, 352 against 338 with 8-bit ones)
    const bool far = n_chunks * kChunk * (state_bits == 8 ? 10 : 16) > ((int64_t)256 << 20);
    const auto kernel = state_bits == 8 ? (far ? adamw_k<8, true> : adamw_k<8, false>) : (far ? adamw_k<32, true> : adamw_k<32, false>);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, a);
    return check_launch("sv_adamw_step");
}

int sv_adamw_decode(const uint8_t* codes, const uint8_t* exponents, float* out, int64_t n, int second, sv_stream_t stream) {
    SV_REQUIRE(n >= 0, "sv_adamw_decode: bad arguments");
    if (n == 0) return SV_OK;
    SV_REQUIRE(codes && exponents && out, "sv_adamw_decode: bad arguments");
    const int64_t n4 = (uintptr_t)codes % 4 == 0 && (uintptr_t)out % 16 == 0 ? n / 4 : 0;
    const dim3 grid((unsigned)ew_grid(n4 > 0 ? n4 : n, 256, 8192));
    const bool far = n * 4 > ((int64_t)256 << 20);
    const auto kernel = second ? (far ? adamw_decode_k<true, true> : adamw_decode_k<true, false>)
                               : (far ? adamw_decode_k<false, true> : adamw_decode_k<false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, to_stream(stream), codes, exponents, out, n, n4);
    return check_launch("sv_adamw_decode");
}

}  // extern "C"
