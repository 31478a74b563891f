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
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at);
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
    if (is_f32) return static_cast<const float *>(base)[at];
    return __uint_as_float((uint32_t)static_cast<const uint16_t *>(base)[at] << 16);
}
__device__ __forceinline__ void store1(void *base, uint64_t at, uint32_t is_f32, float v) {
    if (is_f32) static_cast<float *>(base)[at] = v;
    else static_cast<__nv_bfloat16 *>(base)[at] = __float2bfloat16_rn(v);
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

// Four pairs side by side, from pair number `first` on.
__device__ __forceinline__ void turn_interleaved(float (&v)[8], uint32_t first, uint32_t pairs, const float2 *cs) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (first + j < pairs) {
            const float2 t = cs[first + j];
            const float a = v[2 * j], b = v[2 * j + 1];
            v[2 * j] = a * t.x - b * t.y;
            v[2 * j + 1] = b * t.x + a * t.y;
        }
    }
}

// A block turns `heads` heads of one token; the grid is [tokens][groups of heads]. Bound by memory: a thread takes eight values at a time, or the
// two eights of eight pairs, so that it owns both values of a pair and a call may work in place. (A thread a pair: 36 us for 2048
// tokens of 24 x 256 values, 64 of them turned, fp32 in and bf16 out.)
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p, uint32_t heads) {
    __shared__ float2 cs[kMaxHeadDim / 2];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t = blockIdx.x;
    const uint32_t first_head = blockIdx.y * heads, count = min(heads, p.heads - first_head), pairs = p.rotary.pairs;
    const int32_t position = p.positions[t];
    for (uint32_t i = threadIdx.x; i < pairs; i += blockDim.x) cs[i] = turn(p.rotary, i, position);
    __syncthreads();
    const uint64_t x = t * p.x_stride + (uint64_t)first_head * p.head_dim, o = t * p.out_stride + (uint64_t)first_head * p.head_dim;
    if (p.rotary.interleaved || pairs % 8 == 0) {
        const uint32_t turned = p.rotary.interleaved ? 0 : pairs / 8, per_head = p.head_dim / 8 - turned;  // units of a head; those of two eights come first
#pragma unroll 2
        for (uint32_t u = threadIdx.x; u < count * per_head; u += blockDim.x) {
            const uint32_t h = u / per_head, c = u - h * per_head;
            const uint64_t from = x + (uint64_t)h * p.head_dim, to = o + (uint64_t)h * p.head_dim;
            float a[8], b[8];
            if (c < turned) {
                const uint32_t d = c * 8;
                load8(p.x, from + d, p.x_is_f32, a);
                load8(p.x, from + d + pairs, p.x_is_f32, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 w = cs[d + j];
                    const float va = a[j], vb = b[j];
                    a[j] = va * w.x - vb * w.y;
                    b[j] = vb * w.x + va * w.y;
                }
                store8(p.out, to + d, p.out_is_f32, a);
                store8(p.out, to + d + pairs, p.out_is_f32, b);
            } else {
                const uint32_t d = (c + turned) * 8;
                load8(p.x, from + d, p.x_is_f32, a);
                if (p.rotary.interleaved) turn_interleaved(a, d / 2, pairs, cs);
                store8(p.out, to + d, p.out_is_f32, a);
            }
        }
        return;
    }
    // halves that do not begin at a multiple of eight values: a thread a pair, or a value that is not turned
    const uint32_t per_head = p.head_dim - pairs;
    for (uint32_t u = threadIdx.x; u < count * per_head; u += blockDim.x) {
        const uint32_t h = u / per_head, i = u - h * per_head;
        const uint64_t from = x + (uint64_t)h * p.head_dim + i, to = o + (uint64_t)h * p.head_dim + i;
        float a, b = 0.f;
        if (i < pairs) {
            const float2 c = cs[i];
            const float va = load1(p.x, from, p.x_is_f32), vb = load1(p.x, from + pairs, p.x_is_f32);
            a = va * c.x - vb * c.y;
            b = vb * c.x + va * c.y;
        } else {
            a = load1(p.x, from + pairs, p.x_is_f32);
        }
        if (i < pairs) store1(p.out, to, p.out_is_f32, a);
        store1(p.out, to + pairs, p.out_is_f32, i < pairs ? b : a);
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
    int32_t position, sequence;
    uint32_t page, slot;  // page ~0: padded, or outside the cache
};

__device__ __forceinline__ int32_t sequence_of(const KvTokensParams &p, uint64_t t) { return p.sequences ? p.sequences[t] : (int32_t)(t / p.run); }

__device__ __forceinline__ Place place_of(const KvTokensParams &p, uint64_t t) {
    Place a;
    a.page = ~0u;
    a.slot = 0;
    a.position = p.positions[t];
    a.sequence = sequence_of(p, t);
    if (a.position < 0) return a;
    const uint32_t entry = (uint32_t)a.position / p.kv.page_tokens;
    if ((uint32_t)a.sequence < p.kv.sequences && entry < p.kv.per_sequence) {
        a.slot = (uint32_t)a.position % p.kv.page_tokens;
        const uint32_t page = (uint32_t)p.kv.table[(uint64_t)a.sequence * p.kv.row_stride + entry];
        if (page < p.kv.pages) a.page = page;
    }
    if (a.page == ~0u) *p.kv.input_error = 1;
    return a;
}

__device__ __forceinline__ uint64_t row_offset(const KvView &kv, const Place &a, uint32_t head) {
    return (uint64_t)a.page * kv.page_stride + (uint64_t)head * kv.head_stride + (uint64_t)a.slot * kv.token_stride;
}
__device__ __forceinline__ uint64_t scale_index(const KvView &kv, const Place &a, uint32_t head) {
    return ((uint64_t)a.page * kv.kv_heads + head) * kv.page_tokens + a.slot;
}

// Rows of a block's tokens: keys and values of every head. Each has LANES lanes, eight values a lane; a warp takes 32 / LANES rows at a time.
struct Row {
    uint32_t token, head;  // token of the block
    bool values;
};
__device__ __forceinline__ Row row_of(uint32_t r, uint32_t kv_heads) {
    const uint32_t t = r / (2 * kv_heads), i = r - t * 2 * kv_heads;
    return {t, i < kv_heads ? i : i - kv_heads, i >= kv_heads};
}

constexpr uint32_t kMostTokens = 8;  // of a block

// A block writes up to kMostTokens tokens. Of several tokens with the same place the last one is kept: every block looks through the tokens
// behind its own (most by one comparison with the range of its positions) while its first rows are on their way. Bound by memory for long
// prompts, by latency for single tokens. (A block a token, whole warps for rows of any length: 27 us for 4096 tokens of
// 2 x 4 x 256 fp32 values.)
template <int LANES>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvTokensParams p, uint32_t block_tokens) {
    __shared__ float2 cs[kMostTokens][kMaxHeadDim / 2];
    __shared__ Place places[kMostTokens];
    __shared__ uint32_t replaced;  // a bit a token: one behind it has the same place
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t0 = (uint64_t)blockIdx.x * block_tokens;
    const uint32_t tokens = (uint32_t)min((uint64_t)block_tokens, p.tokens - t0);
    if (threadIdx.x == 0) replaced = 0;
    if (threadIdx.x < tokens) places[threadIdx.x] = place_of(p, t0 + threadIdx.x);
    __syncthreads();
    if (p.rotary.step && p.k_in)
        for (uint32_t i = threadIdx.x; i < tokens * p.rotary.pairs; i += blockDim.x) {
            const uint32_t t = i / p.rotary.pairs;
            cs[t][i - t * p.rotary.pairs] = turn(p.rotary, i - t * p.rotary.pairs, places[t].position);
        }
    int32_t low = 0x7fffffff, high = -1;
    for (uint32_t t = 0; t < tokens; ++t)
        if (places[t].page != ~0u) low = min(low, places[t].position), high = max(high, places[t].position);
#pragma unroll 8
    for (uint64_t u = t0 + 1 + threadIdx.x; u < p.tokens; u += blockDim.x) {
        const int32_t position = p.positions[u];
        if (position >= low && position <= high)
            for (uint32_t t = 0; t < tokens; ++t)
                if (position == places[t].position && u > t0 + t && sequence_of(p, u) == places[t].sequence) atomicOr(&replaced, 1u << t);
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31u, part = lane % LANES, d = part * 8u, rows = tokens * 2 * p.kv.kv_heads;
    const bool has = d < p.kv.head_dim;
#pragma unroll 2
    for (uint32_t r0 = (threadIdx.x >> 5) * (32 / LANES); r0 < rows; r0 += (blockDim.x >> 5) * (32 / LANES)) {
        const uint32_t r = r0 + lane / LANES;
        const Row row = row_of(min(r, rows - 1), p.kv.kv_heads);
        const void *in = row.values ? p.v_in : p.k_in;
        const Place a = places[row.token];
        const bool writes = r < rows && in && a.page != ~0u && !(replaced >> row.token & 1u);
        const uint64_t at = (t0 + row.token) * (row.values ? p.v_stride : p.k_stride) + (uint64_t)row.head * p.kv.head_dim;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (writes && has) load8(in, at + d, p.is_f32, v);
        if (p.rotary.step && p.k_in) {
            const bool turns = writes && !row.values && d < 2 * p.rotary.pairs;
            if (p.rotary.interleaved) {
                if (turns) turn_interleaved(v, d / 2, p.rotary.pairs, cs[row.token]);
            } else if (p.rotary.pairs % 8 == 0) {
                // the other values of the pairs are those of a lane of the same row
                const uint32_t step = p.rotary.pairs / 8, other = (lane & ~(LANES - 1u)) + (part < step ? part + step : part - step) % LANES;
                const uint32_t i = part < step ? d : d - p.rotary.pairs;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float b = __shfl_sync(0xffffffffu, v[j], other);
                    if (turns) v[j] = v[j] * cs[row.token][i + j].x + (part < step ? -b : b) * cs[row.token][i + j].y;
                }
            } else if (turns) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t e = d + j, pairs = p.rotary.pairs;
                    if (e < pairs) v[j] = v[j] * cs[row.token][e].x - load1(in, at + e + pairs, p.is_f32) * cs[row.token][e].y;
                    else if (e < 2 * pairs) v[j] = v[j] * cs[row.token][e - pairs].x + load1(in, at + e - pairs, p.is_f32) * cs[row.token][e - pairs].y;
                }
            }
        }
        uint8_t *const to = (row.values ? p.kv.v : p.kv.k) + (writes ? row_offset(p.kv, a, row.head) : 0);
        if (p.kv.format == 0u) {
            if (writes && has) *reinterpret_cast<uint4 *>(to + 2 * d) = pack8_bf16(v);
            continue;
        }
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        const bool finite = amax < 0x7f800000u;
        const float scale = finite ? __fdiv_rn(__uint_as_float(amax), p.kv.format == 1u ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
        const Divisor by(scale);
        if (writes && has) *reinterpret_cast<uint2 *>(to + d) = finite ? encode8(v, p.kv.format, by) : make_uint2(0u, 0u);
        if (writes && part == 0) (row.values ? p.kv.v_scales : p.kv.k_scales)[scale_index(p.kv, a, row.head)] = scale;
    }
}

template <int LANES>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvTokensParams p, uint32_t block_tokens) {
    __shared__ Place places[kMostTokens];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t0 = (uint64_t)blockIdx.x * block_tokens;
    const uint32_t tokens = (uint32_t)min((uint64_t)block_tokens, p.tokens - t0);
    if (threadIdx.x < tokens) places[threadIdx.x] = place_of(p, t0 + threadIdx.x);
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31u, d = lane % LANES * 8u, rows = tokens * 2 * p.kv.kv_heads;
    if (d >= p.kv.head_dim) return;
#pragma unroll 4
    for (uint32_t r = (threadIdx.x >> 5) * (32 / LANES) + lane / LANES; r < rows; r += (blockDim.x >> 5) * (32 / LANES)) {
        const Row row = row_of(r, p.kv.kv_heads);
        void *out = row.values ? p.v_out : p.k_out;
        const Place a = places[row.token];
        if (!out || a.page == ~0u) continue;
        const uint8_t *from = (row.values ? p.kv.v : p.kv.k) + row_offset(p.kv, a, row.head);
        float v[8];
        if (p.kv.format == 0u) load8(from, d, 0u, v);
        else decode8(*reinterpret_cast<const uint2 *>(from + d), p.kv.format, (row.values ? p.kv.v_scales : p.kv.k_scales)[scale_index(p.kv, a, row.head)], v);
        store8(out, (t0 + row.token) * (row.values ? p.v_stride : p.k_stride) + (uint64_t)row.head * p.kv.head_dim + d, p.is_f32, v);
    }
}

// Tokens of a block: few tokens go to as many blocks as there are, many in eights.
uint32_t block_tokens(uint64_t tokens, uint32_t sm_count) { return (uint32_t)(tokens / (4ull * sm_count) < kMostTokens ? tokens / (4ull * sm_count) + 1 : kMostTokens); }

template <typename Kernel>
cudaError_t launch_tokens(Kernel lanes8, Kernel lanes16, Kernel lanes32, const KvTokensParams &p, uint32_t sm_count, cudaStream_t stream) {
    const uint32_t each = block_tokens(p.tokens, sm_count);
    const Kernel kernel = p.kv.head_dim <= 64 ? lanes8 : p.kv.head_dim <= 128 ? lanes16 : lanes32;
    return launch_dependent(kernel, dim3((uint32_t)((p.tokens + each - 1) / each)), 256, 0, stream, p, each);
}

}  // namespace q4

extern "C" cudaError_t q4k_rotary(const q4::RotaryParams *p, uint32_t sm_count, cudaStream_t stream) {
    // heads of a block: all of a token, or fewer where there are few tokens
    const uint64_t blocks = 2ull * sm_count / p->tokens;
    const uint32_t groups = blocks < 1 ? 1 : blocks > p->heads ? p->heads : (uint32_t)blocks, heads = (p->heads + groups - 1) / groups;
    return q4::launch_dependent(q4::rotary_kernel, dim3((uint32_t)p->tokens, (p->heads + heads - 1) / heads), 256, 0, stream, *p, heads);
}

extern "C" cudaError_t q4k_kv_write(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream) {
    return q4::launch_tokens(q4::kv_write_kernel<8>, q4::kv_write_kernel<16>, q4::kv_write_kernel<32>, *p, sm_count, stream);
}

extern "C" cudaError_t q4k_kv_read(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream) {
    return q4::launch_tokens(q4::kv_read_kernel<8>, q4::kv_read_kernel<16>, q4::kv_read_kernel<32>, *p, sm_count, stream);
}
