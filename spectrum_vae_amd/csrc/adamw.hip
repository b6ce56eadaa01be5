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
#include <algorithm>
#include <new>
#include <vector>

#include "common.h"

namespace sv {
namespace {

constexpr int kBlock = 256;        // elements of an 8-bit block
constexpr int kChunk = 4096;       // elements of one tensor that a workgroup updates at a time
constexpr int kNormParts = 1024;   // most workgroups (partial sums) of the norm launch

struct Tensor {  // one entry of the device table
    float* theta;
    float* grad;
    void* m;
    void* v;
    uint8_t* m_exp;
    uint8_t* v_exp;
    __bf16* theta_lp;
    int64_t n;
    int64_t first_block;  // of its 8-bit blocks among all tensors' (the position in the random stream)
    float decay;
    int32_t vec;          // every pointer takes 4-element accesses
};
struct Chunk {
    int32_t tensor, index;
};
// device image: Tensor[n_tensors], Chunk[n_chunks]

struct StepArgs {
    const Tensor* tensors;
    const Chunk* chunks;
    int64_t n_chunks;
    int64_t* state;
    const double* norm_parts;
    double lr0, log_beta1, log_beta2, log_rate;
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, grad_scale, clip;
    int decay_steps, staircase, zero_grad, n_norm_parts;
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

__device__ __forceinline__ void update(float& th, float& m, float& v, float g, const StepArgs& a, float scale, float alpha,
                                       float lr_decay) {
#pragma clang fp contract(off)
    const float gs = g * scale;
    m = a.beta1 * m + a.one_minus_beta1 * gs;
    v = a.beta2 * v + a.one_minus_beta2 * (gs * gs);
    th = th - lr_decay * th;
    th = th - (alpha * m) / (sqrtf(v) + a.eps);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

// Partial sums of squares of the gradients, one a workgroup, in f64.
__global__ __launch_bounds__(256) void grad_norm_k(const Tensor* __restrict__ tensors, const Chunk* __restrict__ chunks,
                                                    int64_t n_chunks, double* __restrict__ parts) {
    __shared__ double red[4];
    double sum = 0.0;
    for (int64_t k = blockIdx.x; k < n_chunks; k += gridDim.x) {
        const Chunk ck = chunks[k];
        const Tensor& t = tensors[ck.tensor];
        const int64_t i0 = (int64_t)ck.index * kChunk;
        const int n = (int)(t.n - i0 < kChunk ? t.n - i0 : kChunk);
        const float* g = t.grad + i0;
        float s = 0.f;
        for (int i = threadIdx.x; i < n; i += 256) s = fmaf(g[i], g[i], s);
        sum += (double)s;
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// A wave takes blocks of 256 elements, four a lane.
template <int BITS>
__global__ __launch_bounds__(256) void adamw_k(StepArgs a) {
    __shared__ float s_alpha, s_lr, s_scale;
    __shared__ double red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t it = a.state[0];
    double norm2 = 0.0;
    if (a.n_norm_parts > 0) {
        for (int i = threadIdx.x; i < a.n_norm_parts; i += 256) norm2 += a.norm_parts[i];
        for (int o = 32; o > 0; o >>= 1) norm2 += __shfl_xor(norm2, o, 64);
        if (lane == 0) red[wave] = norm2;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        double lr = a.lr0;
        if (a.decay_steps > 0) {
            double e = (double)it / (double)a.decay_steps;
            if (a.staircase) e = floor(e);
            lr *= exp(e * a.log_rate);
        }
        const double t = (double)(it + 1);
        s_alpha = (float)(lr * sqrt(-expm1(t * a.log_beta2)) / -expm1(t * a.log_beta1));
        s_lr = (float)lr;
        float scale = a.grad_scale;
        if (a.n_norm_parts > 0) {
            const double norm = fabs((double)a.grad_scale) * sqrt(red[0] + red[1] + red[2] + red[3]);
            // a norm that is not finite leaves nothing finite, as the clip of Keras
            const float clip = norm > a.clip ? (float)((double)a.clip / norm) : 1.f;
            scale = norm - norm == 0.0 ? a.grad_scale * clip : __uint_as_float(0x7fc00000u);
        }
        s_scale = scale;
    }
    __syncthreads();
    const float alpha = s_alpha, lr = s_lr, scale = s_scale;
    const uint64_t key = mix64(mix64((uint64_t)it) ^ a.seed);
    for (int64_t k = blockIdx.x; k < a.n_chunks; k += gridDim.x) {
        const Chunk ck = a.chunks[k];
        const Tensor t = a.tensors[ck.tensor];
        const float lr_decay = lr * t.decay;
        for (int b = wave; b < kChunk / kBlock; b += 4) {
            const int64_t i0 = (int64_t)ck.index * kChunk + b * kBlock;
            if (i0 >= t.n) break;
            const int64_t i = i0 + 4 * lane;
            const int mine = t.n - i >= 4 ? 4 : t.n - i > 0 ? (int)(t.n - i) : 0;
            float th[4], g[4], m[4], v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                th[e] = e < mine ? t.theta[i + e] : 0.f;
                g[e] = e < mine ? t.grad[i + e] : 0.f;
            }
            const int64_t block = i0 / kBlock;
            if (BITS == 8) {
                const int me = t.m_exp[block], ve = t.v_exp[block];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m[e] = e < mine ? first_value(((const uint8_t*)t.m)[i + e], me) : 0.f;
                    v[e] = e < mine ? second_value(((const uint8_t*)t.v)[i + e], ve) : 0.f;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m[e] = e < mine ? ((const float*)t.m)[i + e] : 0.f;
                    v[e] = e < mine ? ((const float*)t.v)[i + e] : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < mine) update(th[e], m[e], v[e], g[e], a, scale, alpha, lr_decay);
            if (BITS == 8) {
                uint32_t ml = 0, vl = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t mb = __float_as_uint(m[e]) & 0x7fffffffu, vb = __float_as_uint(v[e]) & 0x7fffffffu;
                    ml = mb > ml ? mb : ml;
                    vl = vb > vl ? vb : vl;
                }
                const int me = block_exponent(wave_max(ml)), ve = block_exponent(wave_max(vl));
                const uint64_t pair = (uint64_t)((t.first_block + block) * (kBlock / 2) + 2 * lane);
                const uint64_t h0 = mix64(pair ^ key), h1 = mix64((pair + 1) ^ key);
                const uint32_t r[4] = {(uint32_t)h0, (uint32_t)(h0 >> 32), (uint32_t)h1, (uint32_t)(h1 >> 32)};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < mine) {
                        ((uint8_t*)t.m)[i + e] = (uint8_t)first_code(m[e], me, r[e] & 0xffffu);
                        ((uint8_t*)t.v)[i + e] = (uint8_t)second_code(v[e], ve, r[e] >> 16);
                    }
                if (lane == 0) {
                    t.m_exp[block] = (uint8_t)me;
                    t.v_exp[block] = (uint8_t)ve;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < mine) {
                        ((float*)t.m)[i + e] = m[e];
                        ((float*)t.v)[i + e] = v[e];
                    }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < mine) {
                    t.theta[i + e] = th[e];
                    if (t.theta_lp != nullptr) t.theta_lp[i + e] = (__bf16)th[e];
                    if (a.zero_grad) t.grad[i + e] = 0.f;
                }
        }
    }
    // the workgroup that arrives last advances the count: every workgroup has read it by then
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned int* ticket = reinterpret_cast<unsigned int*>(a.state + 2);
        const unsigned int prev = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (prev == gridDim.x - 1) {
            a.state[0] = it + 1;
            reinterpret_cast<float*>(a.state + 1)[0] = alpha;
            reinterpret_cast<float*>(a.state + 1)[1] = lr;
            __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

template <bool SECOND>
__global__ __launch_bounds__(256) void adamw_decode_k(const uint8_t* __restrict__ code, const uint8_t* __restrict__ exps,
                                                       float* __restrict__ out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
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
    return (size_t)n_tensors * sizeof(Tensor) + (size_t)*n_chunks * sizeof(Chunk);
}

int sv_adamw_plan_fill(const sv_adamw_tensor* tensors, int n_tensors, int state_bits, void* image, size_t image_bytes) {
    try {
        int rc = plan_check("sv_adamw_plan_fill", tensors, n_tensors, state_bits);
        if (rc) return rc;
        int64_t n_chunks = 0;
        const size_t need = sv_adamw_plan_bytes(tensors, n_tensors, &n_chunks);
        if (image == nullptr || image_bytes < need)
            return fail(SV_E_WORKSPACE, "sv_adamw_plan_fill: image %zu bytes < required %zu", image_bytes, need);
        Tensor* table = (Tensor*)image;
        Chunk* chunk = (Chunk*)(table + n_tensors);
        int64_t block = 0;
        for (int i = 0; i < n_tensors; ++i) {
            const sv_adamw_tensor& e = tensors[i];
            const uintptr_t state_align = state_bits == 8 ? 4 : 16;
            const bool vec = (uintptr_t)e.theta % 16 == 0 && (uintptr_t)e.grad % 16 == 0 && (uintptr_t)e.m % state_align == 0 &&
                             (uintptr_t)e.v % state_align == 0 && (uintptr_t)e.theta_bf16 % 8 == 0;
            table[i] = Tensor{e.theta, e.grad, e.m, e.v, e.m_exp, e.v_exp, (__bf16*)e.theta_bf16, e.n, block, e.weight_decay, vec};
            block += ceil_div(e.n, kBlock);
            for (int64_t k = 0; k < ceil_div(e.n, kChunk); ++k) *chunk++ = Chunk{i, (int32_t)k};
        }
        return SV_OK;
    } catch (const std::bad_alloc&) {
        return fail(SV_E_INVALID, "sv_adamw_plan_fill: out of host memory");
    }
}

size_t sv_adamw_workspace_bytes(void) { return kNormParts * sizeof(double); }

int sv_adamw_step(const void* plan, int n_tensors, int64_t n_chunks, int state_bits, int64_t* step_state, double lr0,
                  double beta1, double beta2, float eps, int decay_steps, double decay_rate, int staircase, float grad_scale,
                  float clip_norm, uint64_t seed, int zero_grad, void* workspace, size_t workspace_bytes, sv_stream_t stream) {
    SV_REQUIRE(plan != nullptr && step_state != nullptr && n_tensors >= 1 && n_chunks >= 0, "sv_adamw_step: bad arguments");
    SV_REQUIRE((uintptr_t)plan % 8 == 0 && (uintptr_t)step_state % 8 == 0, "sv_adamw_step: plan / state must be 8-byte aligned");
    SV_REQUIRE(state_bits == 8 || state_bits == 32, "sv_adamw_step: moments have 8 or 32 bits, not %d", state_bits);
    SV_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "sv_adamw_step: betas out of range");
    SV_REQUIRE(eps > 0.f && clip_norm >= 0.f && (decay_steps <= 0 || decay_rate > 0.0), "sv_adamw_step: epsilon and the decay rate must be positive, the clip not negative");
    SV_REQUIRE(clip_norm == 0.f || (workspace != nullptr && (uintptr_t)workspace % 8 == 0), "sv_adamw_step: clipping needs a workspace");
    if (clip_norm > 0.f && workspace_bytes < sv_adamw_workspace_bytes())
        return fail(SV_E_WORKSPACE, "sv_adamw_step: workspace %zu bytes < required %zu", workspace_bytes, sv_adamw_workspace_bytes());
    hipStream_t st = to_stream(stream);
    StepArgs a{};
    a.tensors = (const Tensor*)plan;
    a.chunks = (const Chunk*)(a.tensors + n_tensors);
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
        hipLaunchKernelGGL(grad_norm_k, dim3(a.n_norm_parts), dim3(256), 0, st, a.tensors, a.chunks, n_chunks, (double*)workspace);
    }
    const int grid = (int)(n_chunks < 1 ? 1 : n_chunks < 2048 ? n_chunks : 2048);
    if (state_bits == 8)
        hipLaunchKernelGGL(adamw_k<8>, dim3(grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(adamw_k<32>, dim3(grid), dim3(256), 0, st, a);
    return check_launch("sv_adamw_step");
}

int sv_adamw_decode(const uint8_t* codes, const uint8_t* exponents, float* out, int64_t n, int second, sv_stream_t stream) {
    SV_REQUIRE(n >= 0, "sv_adamw_decode: bad arguments");
    if (n == 0) return SV_OK;
    SV_REQUIRE(codes && exponents && out, "sv_adamw_decode: bad arguments");
    if (second)
        hipLaunchKernelGGL(adamw_decode_k<true>, dim3(ew_grid(n, 256, 8192)), dim3(256), 0, to_stream(stream), codes, exponents, out, n);
    else
        hipLaunchKernelGGL(adamw_decode_k<false>, dim3(ew_grid(n, 256, 8192)), dim3(256), 0, to_stream(stream), codes, exponents, out, n);
    return check_launch("sv_adamw_decode");
}

}  // extern "C"
