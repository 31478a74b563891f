// Rotary positions, and a paged cache of keys and values that is quantised as it is written. Counterparts in the reference:
// src/metal_runtime.rs:5171-5475, 7298-7457, shaders/qwen38.metal:4761-5323 (rotary preparation, int8 append).
#include "q4_attention.h"

#include <cuda_fp8.h>

#include "q4_device.cuh"

namespace q4 {

// ---- activations: eight values at a time, fp32 or bf16 ----

__device__ __forceinline__ void load8(const void *base, uint64_t at, uint32_t is_f32, float (&v)[8]) {
    if (is_f32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
        const float4 a = __ldcg(p), b = __ldcg(p + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8]) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

__device__ __forceinline__ void store8(void *base, uint64_t at, uint32_t is_f32, const float (&v)[8]) {
    if (is_f32) {
        float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(base) + at);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + at) = pack8_bf16(v);
    }
}

__device__ __forceinline__ float load1(const void *base, uint64_t at, uint32_t is_f32) {
    if (is_f32) return __ldcg(static_cast<const float *>(base) + at);
    return __uint_as_float((uint32_t)__ldcg(static_cast<const uint16_t *>(base) + at) << 16);
}

// ---- rotary ----

// Cosine and sine of pair i at a position. position * step wraps at 2^64, which is one turn, so the product is the angle
// modulo a turn with no error but the step's own (2^-65 turns a token); as a signed number it lies within half a turn, and its
// rounding to 24 bits is relative. A 32-bit product of a position and a frequency would be off by 0.03 rad at position 262144.
__device__ __forceinline__ float2 turn(const RotaryView &r, uint32_t i, int32_t position) {
    const uint64_t phase = (uint64_t)(int64_t)position * r.step[i];
    float s, c;
    sincospif(__ll2float_rn((long long)phase) * 0x1p-63f, &s, &c);
    return make_float2(c * r.factor, s * r.factor);
}

// Eight values of a head from number d on, turned; `at` is the head's first value. Those of the other half of their pairs are
// read again (from L1 or L2, the same head's lines). Pairs in `cs` (shared memory).
__device__ __forceinline__ void load8_turned(const void *x, uint64_t at, uint32_t d, uint32_t is_f32, const RotaryView &r, const float2 *cs, float (&v)[8]) {
    load8(x, at + d, is_f32, v);
    if (d >= 2 * r.pairs) return;
    if (r.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t i = d / 2 + j;
            if (i < r.pairs) {
                const float2 t = cs[i];
                const float a = v[2 * j], b = v[2 * j + 1];
                v[2 * j] = a * t.x - b * t.y;
                v[2 * j + 1] = b * t.x + a * t.y;
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t e = d + j;
        if (e < r.pairs) v[j] = v[j] * cs[e].x - load1(x, at + e + r.pairs, is_f32) * cs[e].y;
        else if (e < 2 * r.pairs) v[j] = v[j] * cs[e - r.pairs].x + load1(x, at + e - r.pairs, is_f32) * cs[e - r.pairs].y;
    }
}

__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
    __shared__ float2 cs[kMaxHeadDim / 2];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t = blockIdx.x;
    const int32_t position = __ldcg(p.positions + t);
    for (uint32_t i = threadIdx.x; i < p.rotary.pairs; i += blockDim.x) cs[i] = turn(p.rotary, i, position);
    __syncthreads();
    // a thread owns both values of a pair, so that a call may work in place
    const uint32_t rest = p.head_dim - 2 * p.rotary.pairs, per_head = p.rotary.pairs + rest;
    for (uint32_t u = threadIdx.x; u < p.heads * per_head; u += blockDim.x) {
        const uint32_t h = u / per_head, i = u % per_head;
        const uint64_t x = t * p.x_stride + (uint64_t)h * p.head_dim, o = t * p.out_stride + (uint64_t)h * p.head_dim;
        uint32_t d0, d1;
        float a, b = 0.f;
        if (i < p.rotary.pairs) {
            d0 = p.rotary.interleaved ? 2 * i : i;
            d1 = p.rotary.interleaved ? 2 * i + 1 : i + p.rotary.pairs;
            const float2 c = cs[i];
            const float va = load1(p.x, x + d0, p.x_is_f32), vb = load1(p.x, x + d1, p.x_is_f32);
            a = va * c.x - vb * c.y;
            b = vb * c.x + va * c.y;
        } else {
            d0 = d1 = i + p.rotary.pairs;
            a = b = load1(p.x, x + d0, p.x_is_f32);
        }
        if (p.out_is_f32) {
            static_cast<float *>(p.out)[o + d0] = a;
            if (d1 != d0) static_cast<float *>(p.out)[o + d1] = b;
        } else {
            static_cast<__nv_bfloat16 *>(p.out)[o + d0] = __float2bfloat16_rn(a);
            if (d1 != d0) static_cast<__nv_bfloat16 *>(p.out)[o + d1] = __float2bfloat16_rn(b);
        }
    }
}

// ---- codes ----

// A code is the number nearest to x / scale, ties to even, for the exact quotient: reading back differs by whole codes where two
// ways to divide disagree, so a product with 1 / scale alone is not enough. Scales below 2^-100 (whose reciprocal or residuals
// leave the range of 32 bits) take a division in 64 bits.
struct Divisor {
    float scale, inverse, half;
    bool tiny;
    __device__ explicit Divisor(float s) : scale(s), inverse(1.0f / s), half(0.5f * s), tiny(s < 0x1p-100f) {}
    // x * (1 / scale) is within 2^-16 of the quotient, so its nearest integer is off by one at most, and the residual
    // x - q * scale, which one fused operation gives exactly, tells.
    __device__ int int8(float x) const {
        if (tiny) return scale > 0.f ? (int)fmin(fmax(rint((double)x / (double)scale), -127.0), 127.0) : 0;
        float q = rintf(x * inverse);
        const float t = fmaf(-q, scale, x);
        const bool odd = ((int)q & 1) != 0;
        if (t > half || (t == half && odd)) q += 1.f;
        else if (t < -half || (t == -half && odd)) q -= 1.f;
        return (int)q;
    }
    // The quotient rounded to odd: to 24 bits towards zero, the last bit set if anything was cut off. Rounding that to the 4 bits
    // of an e4m3 number gives what rounding the exact quotient gives.
    __device__ float odd(float x) const {
        if (tiny) {
            if (!(scale > 0.f)) return 0.f;
            const double q = (double)x / (double)scale;
            const float r = __double2float_rz(q);
            return (double)r == q ? r : __uint_as_float(__float_as_uint(r) | 1u);
        }
        float r = x * inverse;
        r = fmaf(fmaf(-r, scale, x), inverse, r);
        const float e = fmaf(-r, scale, x);  // its sign is exact
        uint32_t bits = __float_as_uint(r);
        if (e == 0.f || r == 0.f) return r;
        if ((__float_as_uint(e) ^ bits) >> 31) bits -= 1u;  // r lies beyond the quotient
        return __uint_as_float(bits | 1u);
    }
};

__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t format, const Divisor &by) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        uint32_t pair;
        if (format == 1u) {
            pair = ((uint32_t)by.int8(v[i]) & 0xffu) | (((uint32_t)by.int8(v[i + 1]) & 0xffu) << 8);
        } else {
            pair = __nv_cvt_float2_to_fp8x2(make_float2(by.odd(v[i]), by.odd(v[i + 1])), __NV_SATFINITE, __NV_E4M3);
        }
        w[i / 4] |= pair << (i % 4 * 8);
    }
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void decode8(uint2 c, uint32_t format, float scale, float (&v)[8]) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t pair = (w[i / 4] >> (i % 4 * 8)) & 0xffffu;
        if (format == 1u) {
            v[i] = (float)(int8_t)(pair & 0xffu) * scale;
            v[i + 1] = (float)(int8_t)(pair >> 8) * scale;
        } else {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            v[i] = f.x * scale;
            v[i + 1] = f.y * scale;
        }
    }
}

// ---- where a token stands ----

struct Place {
    bool there;
    uint32_t sequence, page, slot;
    int32_t position;
};

__device__ __forceinline__ uint32_t sequence_of(const KvTokensParams &p, uint64_t t) {
    return p.sequences ? (uint32_t)__ldcg(p.sequences + t) : (uint32_t)(t / p.run);
}

// (every thread of a block finds the same; one of them reports)
__device__ __forceinline__ Place place_of(const KvTokensParams &p, uint64_t t) {
    Place a;
    a.there = false;
    a.page = a.slot = 0;
    a.position = __ldcg(p.positions + t);
    a.sequence = sequence_of(p, t);
    if (a.position < 0) return a;
    bool bad = a.sequence >= p.kv.sequences;
    if (!bad) {
        const uint32_t entry = (uint32_t)a.position / p.kv.page_tokens;
        bad = entry >= p.kv.per_sequence;
        if (!bad) {
            a.slot = (uint32_t)a.position % p.kv.page_tokens;
            a.page = (uint32_t)__ldcg(p.kv.table + (uint64_t)a.sequence * p.kv.row_stride + entry);
            bad = a.page >= p.kv.pages;
        }
    }
    if (bad && threadIdx.x == 0) *p.kv.input_error = 1;
    a.there = !bad;
    return a;
}

__device__ __forceinline__ uint64_t row_offset(const KvView &kv, const Place &a, uint32_t head) {
    return (uint64_t)a.page * kv.page_stride + (uint64_t)head * kv.head_stride + (uint64_t)a.slot * kv.token_stride;
}
__device__ __forceinline__ uint64_t scale_index(const KvView &kv, const Place &a, uint32_t head) {
    return ((uint64_t)a.page * kv.kv_heads + head) * kv.page_tokens + a.slot;
}

// One block per token, one warp per head of K and of V at a time, eight values a lane.
__global__ void __launch_bounds__(256) kv_write_kernel(const KvTokensParams p) {
    __shared__ float2 cs[kMaxHeadDim / 2];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t = blockIdx.x;
    const Place a = place_of(p, t);
    if (!a.there) return;
    // of several tokens with the same place the last one is kept
    int later = 0;
    for (uint64_t u = t + 1 + threadIdx.x; u < p.tokens; u += blockDim.x) later |= __ldcg(p.positions + u) == a.position && sequence_of(p, u) == a.sequence;
    if (__syncthreads_or(later)) return;
    if (p.rotary.step && p.k_in) {
        for (uint32_t i = threadIdx.x; i < p.rotary.pairs; i += blockDim.x) cs[i] = turn(p.rotary, i, a.position);
        __syncthreads();
    }
    const uint32_t lane = threadIdx.x & 31u, d = lane * 8u;
    const bool has = d < p.kv.head_dim;
    for (uint32_t r = threadIdx.x >> 5; r < 2 * p.kv.kv_heads; r += blockDim.x >> 5) {
        const bool is_k = r < p.kv.kv_heads;
        const uint32_t head = is_k ? r : r - p.kv.kv_heads;
        const void *in = is_k ? p.k_in : p.v_in;
        if (!in) continue;
        const uint64_t at = t * (is_k ? p.k_stride : p.v_stride) + (uint64_t)head * p.kv.head_dim;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (has) {
            if (is_k && p.rotary.step) load8_turned(in, at, d, p.is_f32, p.rotary, cs, v);
            else load8(in, at + d, p.is_f32, v);
        }
        uint8_t *row = (is_k ? p.kv.k : p.kv.v) + row_offset(p.kv, a, head);
        if (p.kv.format == 0u) {
            if (has) *reinterpret_cast<uint4 *>(row + 2 * d) = pack8_bf16(v);
            continue;
        }
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
        amax = __reduce_max_sync(0xffffffffu, amax);
        const bool finite = amax < 0x7f800000u;
        const float scale = finite ? __fdiv_rn(__uint_as_float(amax), p.kv.format == 1u ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
        const Divisor by(scale);
        if (has) *reinterpret_cast<uint2 *>(row + d) = finite ? encode8(v, p.kv.format, by) : make_uint2(0u, 0u);
        if (lane == 0) (is_k ? p.kv.k_scales : p.kv.v_scales)[scale_index(p.kv, a, head)] = scale;
    }
}

__global__ void __launch_bounds__(256) kv_read_kernel(const KvTokensParams p) {
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t = blockIdx.x;
    const Place a = place_of(p, t);
    if (!a.there) return;
    const uint32_t d = (threadIdx.x & 31u) * 8u;
    if (d >= p.kv.head_dim) return;
    for (uint32_t r = threadIdx.x >> 5; r < 2 * p.kv.kv_heads; r += blockDim.x >> 5) {
        const bool is_k = r < p.kv.kv_heads;
        const uint32_t head = is_k ? r : r - p.kv.kv_heads;
        void *out = is_k ? p.k_out : p.v_out;
        if (!out) continue;
        const uint8_t *row = (is_k ? p.kv.k : p.kv.v) + row_offset(p.kv, a, head);
        float v[8];
        if (p.kv.format == 0u) load8(row, d, 0u, v);
        else decode8(__ldcg(reinterpret_cast<const uint2 *>(row + d)), p.kv.format, __ldcg((is_k ? p.kv.k_scales : p.kv.v_scales) + scale_index(p.kv, a, head)), v);
        store8(out, t * (is_k ? p.k_stride : p.v_stride) + (uint64_t)head * p.kv.head_dim + d, p.is_f32, v);
    }
}

}  // namespace q4

extern "C" cudaError_t q4k_rotary(const q4::RotaryParams *p, cudaStream_t stream) {
    return q4::launch_dependent(q4::rotary_kernel, dim3((uint32_t)p->tokens), 256, 0, stream, *p);
}

extern "C" cudaError_t q4k_kv_write(const q4::KvTokensParams *p, cudaStream_t stream) {
    return q4::launch_dependent(q4::kv_write_kernel, dim3((uint32_t)p->tokens), 256, 0, stream, *p);
}

extern "C" cudaError_t q4k_kv_read(const q4::KvTokensParams *p, cudaStream_t stream) {
    return q4::launch_dependent(q4::kv_read_kernel, dim3((uint32_t)p->tokens), 256, 0, stream, *p);
}
