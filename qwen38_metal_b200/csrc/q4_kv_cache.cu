// Rotary positions, and a paged cache of keys and values that is quantised as it is written. Counterparts in the reference:
// src/metal_runtime.rs:5171-5475, 7298-7457, shaders/qwen38.metal:4761-5323 (rotary preparation, int8 append).
#include "q4_attention.h"

#include <cuda_fp8.h>

#include "q4_device.cuh"

namespace q4 {

// ---- activations: eight values at a time, fp32 or bf16 ----

__device__ __forceinline__ void unpack8_bf16(uint4 a, float (&v)[8]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ void load8(const void *base, uint64_t at, uint32_t is_f32, float (&v)[8]) {
    if (is_f32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        unpack8_bf16(*reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at), v);
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
// ways to divide disagree, so a product with 1 / scale alone is not enough.
constexpr float kTinyScale = 0x1p-80f;  // below it reciprocals or residuals leave the range of 32 bits

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }

// The codes of quotients in 64 bits, which rounds no quotient of two 24-bit numbers onto or across the middle between two codes. For e4m3
// the quotient goes to 24 bits towards zero with the last bit set if anything was cut off: rounding that to 4 bits is rounding it.
template <int FMT>
__device__ __noinline__ uint2 encode8_exactly(float4 a, float4 b, float scale) {
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t w[2] = {0u, 0u};
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        const double q = scale > 0.f ? (double)v[i] / (double)scale : 0.0;
        uint32_t code;
        if (FMT == 1) {
            code = (uint32_t)(int)fmin(fmax(rint(q), -127.0), 127.0) & 0xffu;
        } else {
            const float r = __double2float_rz(q);
            code = e4m3_pair((double)r == q ? r : __uint_as_float(__float_as_uint(r) | 1u), 0.f) & 0xffu;
        }
        if (i < 4) w[0] |= code << (i * 8);
        else w[1] |= code << (i * 8 - 32);
    }
    return make_uint2(w[0], w[1]);
}

// int8: x * (1 / scale) is within 2^-22 of the quotient (relative). Where that could be on the other side of the middle between two codes, all
// eight are done exactly: seldom (one in 10^5 values). e4m3: the middles are numbers of 5 bits, and bf16 values meet them often (every fourth
// row has one: 3/4 of an even largest value, for one). So the product goes to the nearest number m of 5 bits; the sign of x - m * scale is
// exact, and the number given to the conversion is on that side of m, or m itself.
template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float scale) {
    const float inverse = 1.0f / scale;
    bool sure = scale >= kTinyScale;
    uint32_t w[2];
    if (FMT == 1) {
        // 1.5 * 2^23 + quotient: the sum is rounded to a whole number, whose low byte is the code. x - q * scale is exact.
        uint32_t n[8];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = fmaf(v[i], inverse, 12582912.f);
            most = fmaxf(most, fabsf(fmaf(12582912.f - m, scale, v[i])));
            n[i] = __float_as_uint(m);
        }
        sure = sure && most < 0.5f * scale;
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = __byte_perm(__byte_perm(n[4 * i], n[4 * i + 1], 0x0040), __byte_perm(n[4 * i + 2], n[4 * i + 3], 0x0040), 0x5410);
    } else {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = __uint_as_float(__float_as_uint(v[i] * inverse) + 0x40000u & 0xfff80000u), r = fmaf(-m, scale, v[i]);
            q[i] = __fmaf_rz(r, inverse, m);
            if (r != 0.f) q[i] = __uint_as_float(__float_as_uint(q[i]) | 1u);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = e4m3_pair(q[4 * i], q[4 * i + 1]) | e4m3_pair(q[4 * i + 2], q[4 * i + 3]) << 16;
    }
    if (!sure) return encode8_exactly<FMT>(make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]), scale);
    return make_uint2(w[0], w[1]);
}

template <int FMT>
__device__ __forceinline__ void decode8(uint2 c, float scale, float (&v)[8]) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t pair = (w[i / 4] >> (i % 4 * 8)) & 0xffffu;
        if (FMT == 1) {
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
constexpr uint32_t kRowsAhead = 4;   // rows that are on their way to a lane

// A block writes up to kMostTokens tokens. Of several tokens with the same place the last one is kept: every block looks through the tokens
// behind its own (most by one comparison with the range of its positions) while its first rows are on their way. Bound by memory for long
// prompts, by latency for single tokens. (A block a token, whole warps for rows of any length: 27 us for 4096 tokens of
// 2 x 4 x 256 fp32 values.)
template <int FMT, int LANES, bool TURN>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvTokensParams p, uint32_t block_tokens) {
    __shared__ float2 cs[TURN ? kMostTokens : 1][kMaxHeadDim / 2];
    __shared__ Place places[kMostTokens];
    __shared__ uint32_t replaced;  // a bit a token: one behind it has the same place
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t0 = (uint64_t)blockIdx.x * block_tokens;
    const uint32_t tokens = (uint32_t)min((uint64_t)block_tokens, p.tokens - t0), pairs = p.rotary.pairs;
    const uint32_t lane = threadIdx.x & 31u, part = lane % LANES, d = part * 8u, rows = tokens * 2 * p.kv.kv_heads;
    const uint32_t step = (blockDim.x >> 5) * (32 / LANES);
    float v[kRowsAhead][8];
    uint32_t r0 = (threadIdx.x >> 5) * (32 / LANES);
    const auto load_rows = [&]() {
#pragma unroll
        for (uint32_t k = 0; k < kRowsAhead; ++k) {
            const uint32_t r = r0 + k * step + lane / LANES;
            const Row row = row_of(min(r, rows - 1), p.kv.kv_heads);
            const void *in = row.values ? p.v_in : p.k_in;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
            if (r < rows && in && d < p.kv.head_dim) load8(in, (t0 + row.token) * (row.values ? p.v_stride : p.k_stride) + (uint64_t)row.head * p.kv.head_dim + d, p.is_f32, v[k]);
        }
    };
    load_rows();
    if (threadIdx.x == 0) replaced = 0;
    if (threadIdx.x < tokens) places[threadIdx.x] = place_of(p, t0 + threadIdx.x);
    __syncthreads();
    if (TURN)
        for (uint32_t i = threadIdx.x; i < tokens * pairs; i += blockDim.x) {
            const uint32_t t = i / pairs;
            cs[t][i - t * pairs] = turn(p.rotary, i - t * pairs, places[t].position);
        }
    int32_t low = 0x7fffffff, high = -1;
    for (uint32_t t = 0; t < tokens; ++t)
        if (places[t].page != ~0u) low = min(low, places[t].position), high = max(high, places[t].position);
    const auto compare = [&](uint64_t u, int32_t position) {
        if (position >= low && position <= high)
#pragma unroll 1
            for (uint32_t t = 0; t < tokens; ++t)
                if (position == places[t].position && u > t0 + t && sequence_of(p, u) == places[t].sequence) atomicOr(&replaced, 1u << t);
    };
    // the tokens behind the block's first, four at a time from the first whose position starts at 16 bytes
    const uint64_t behind = t0 + 1, fours = min(p.tokens, behind + (0u - (uint32_t)((uintptr_t)(p.positions + behind) >> 2) & 3u)), last = fours + ((p.tokens - min(fours, p.tokens)) & ~3ull);
    if (threadIdx.x < fours - min(behind, fours)) compare(behind + threadIdx.x, p.positions[behind + threadIdx.x]);
    if (threadIdx.x < p.tokens - last) compare(last + threadIdx.x, p.positions[last + threadIdx.x]);
#pragma unroll 2
    for (uint64_t u = fours + 4 * threadIdx.x; u < last; u += 4 * blockDim.x) {
        const int4 position = *reinterpret_cast<const int4 *>(p.positions + u);
        if (min(min(position.x, position.y), min(position.z, position.w)) <= high && max(max(position.x, position.y), max(position.z, position.w)) >= low) {
            compare(u, position.x);
            compare(u + 1, position.y);
            compare(u + 2, position.z);
            compare(u + 3, position.w);
        }
    }
    __syncthreads();
#pragma unroll 1
    for (;;) {
#pragma unroll
        for (uint32_t k = 0; k < kRowsAhead; ++k) {
            const uint32_t r = r0 + k * step + lane / LANES;
            if (r0 + k * step >= rows) break;
            const Row row = row_of(min(r, rows - 1), p.kv.kv_heads);
            const Place a = places[row.token];
            const bool writes = r < rows && (row.values ? p.v_in : p.k_in) && a.page != ~0u && !(replaced >> row.token & 1u);
            if (TURN) {
                const bool turns = !row.values && d < 2 * pairs;
                if (p.rotary.interleaved) {
                    if (turns) turn_interleaved(v[k], d / 2, pairs, cs[row.token]);
                } else if (pairs % 8 == 0) {
                    // the other values of the pairs are those of a lane of the same row
                    const uint32_t by = pairs / 8, other = (lane & ~(LANES - 1u)) + (part < by ? part + by : part - by) % LANES;
                    const uint32_t i = part < by ? d : d - pairs;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float b = __shfl_sync(0xffffffffu, v[k][j], other);
                        if (turns) v[k][j] = v[k][j] * cs[row.token][i + j].x + (part < by ? -b : b) * cs[row.token][i + j].y;
                    }
                } else if (turns && writes) {
                    const uint64_t at = (t0 + row.token) * p.k_stride + (uint64_t)row.head * p.kv.head_dim;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t e = d + j;
                        if (e < pairs) v[k][j] = v[k][j] * cs[row.token][e].x - load1(p.k_in, at + e + pairs, p.is_f32) * cs[row.token][e].y;
                        else if (e < 2 * pairs) v[k][j] = v[k][j] * cs[row.token][e - pairs].x + load1(p.k_in, at + e - pairs, p.is_f32) * cs[row.token][e - pairs].y;
                    }
                }
            }
            uint8_t *const to = (row.values ? p.kv.v : p.kv.k) + (writes ? row_offset(p.kv, a, row.head) : 0);
            const bool has = writes && d < p.kv.head_dim;
            if (FMT == 0) {
                if (has) *reinterpret_cast<uint4 *>(to + 2 * d) = pack8_bf16(v[k]);
                continue;
            }
            uint32_t amax = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[k][j]) & 0x7fffffffu);
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
            const bool finite = amax < 0x7f800000u;
            const float scale = finite ? __fdiv_rn(__uint_as_float(amax), FMT == 1 ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
            if (has) *reinterpret_cast<uint2 *>(to + d) = finite ? encode8<FMT == 0 ? 1 : FMT>(v[k], scale) : make_uint2(0u, 0u);
            if (writes && part == 0) (row.values ? p.kv.v_scales : p.kv.k_scales)[scale_index(p.kv, a, row.head)] = scale;
        }
        r0 += kRowsAhead * step;
        if (r0 >= rows) break;
        load_rows();
    }
}

template <int FMT, int LANES>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvTokensParams p, uint32_t block_tokens) {
    __shared__ Place places[kMostTokens];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t0 = (uint64_t)blockIdx.x * block_tokens;
    const uint32_t tokens = (uint32_t)min((uint64_t)block_tokens, p.tokens - t0);
    if (threadIdx.x < tokens) places[threadIdx.x] = place_of(p, t0 + threadIdx.x);
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31u, d = lane % LANES * 8u, rows = tokens * 2 * p.kv.kv_heads, step = (blockDim.x >> 5) * (32 / LANES);
    if (d >= p.kv.head_dim) return;
#pragma unroll 1
    for (uint32_t r0 = (threadIdx.x >> 5) * (32 / LANES) + lane / LANES; r0 < rows; r0 += kRowsAhead * step) {
        uint4 held[kRowsAhead];
        float scale[kRowsAhead];
        bool there[kRowsAhead];
#pragma unroll
        for (uint32_t k = 0; k < kRowsAhead; ++k) {
            const uint32_t r = r0 + k * step;
            const Row row = row_of(min(r, rows - 1), p.kv.kv_heads);
            const Place a = places[row.token];
            there[k] = r < rows && (row.values ? p.v_out : p.k_out) && a.page != ~0u;
            held[k] = make_uint4(0u, 0u, 0u, 0u);
            scale[k] = 1.f;
            if (!there[k]) continue;
            const uint8_t *from = (row.values ? p.kv.v : p.kv.k) + row_offset(p.kv, a, row.head);
            if (FMT == 0) {
                held[k] = *reinterpret_cast<const uint4 *>(from + 2 * d);
            } else {
                const uint2 c = *reinterpret_cast<const uint2 *>(from + d);
                held[k].x = c.x, held[k].y = c.y;
                scale[k] = (row.values ? p.kv.v_scales : p.kv.k_scales)[scale_index(p.kv, a, row.head)];
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kRowsAhead; ++k) {
            if (!there[k]) continue;
            const Row row = row_of(r0 + k * step, p.kv.kv_heads);
            float v[8];
            if (FMT == 0) unpack8_bf16(held[k], v);
            else decode8<FMT == 0 ? 1 : FMT>(make_uint2(held[k].x, held[k].y), scale[k], v);
            store8(row.values ? p.v_out : p.k_out, (t0 + row.token) * (row.values ? p.v_stride : p.k_stride) + (uint64_t)row.head * p.kv.head_dim + d, p.is_f32, v);
        }
    }
}

// Tokens of a block: few tokens go to as many blocks as there are, many in eights.
uint32_t block_tokens(uint64_t tokens, uint32_t sm_count) { return (uint32_t)(tokens / (8ull * sm_count) < kMostTokens ? tokens / (8ull * sm_count) + 1 : kMostTokens); }

template <int FMT, int LANES>
cudaError_t launch_tokens(const KvTokensParams &p, bool write, uint32_t sm_count, cudaStream_t stream) {
    const uint32_t each = block_tokens(p.tokens, sm_count);
    const auto kernel = !write ? kv_read_kernel<FMT, LANES> : p.rotary.step && p.k_in ? kv_write_kernel<FMT, LANES, true> : kv_write_kernel<FMT, LANES, false>;
    return launch_dependent(kernel, dim3((uint32_t)((p.tokens + each - 1) / each)), 256, 0, stream, p, each);
}

template <int FMT>
cudaError_t launch_tokens(const KvTokensParams &p, bool write, uint32_t sm_count, cudaStream_t stream) {
    if (p.kv.head_dim <= 64) return launch_tokens<FMT, 8>(p, write, sm_count, stream);
    if (p.kv.head_dim <= 128) return launch_tokens<FMT, 16>(p, write, sm_count, stream);
    return launch_tokens<FMT, 32>(p, write, sm_count, stream);
}

cudaError_t launch_tokens(const KvTokensParams &p, bool write, uint32_t sm_count, cudaStream_t stream) {
    if (p.kv.format == 0u) return launch_tokens<0>(p, write, sm_count, stream);
    if (p.kv.format == 1u) return launch_tokens<1>(p, write, sm_count, stream);
    return launch_tokens<2>(p, write, sm_count, stream);
}

}  // namespace q4

extern "C" cudaError_t q4k_rotary(const q4::RotaryParams *p, uint32_t sm_count, cudaStream_t stream) {
    // heads of a block: all of a token, or fewer where there are few tokens
    const uint64_t blocks = 2ull * sm_count / p->tokens;
    const uint32_t groups = blocks < 1 ? 1 : blocks > p->heads ? p->heads : (uint32_t)blocks, heads = (p->heads + groups - 1) / groups;
    return q4::launch_dependent(q4::rotary_kernel, dim3((uint32_t)p->tokens, (p->heads + heads - 1) / heads), 256, 0, stream, *p, heads);
}

extern "C" cudaError_t q4k_kv_write(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream) {
    return q4::launch_tokens(*p, true, sm_count, stream);
}

extern "C" cudaError_t q4k_kv_read(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream) {
    return q4::launch_tokens(*p, false, sm_count, stream);
}
