// Rotary positions, and a paged cache of keys and values that is quantised as it is written. Counterparts in the reference:
// src/metal_runtime.rs:5171-5475, 7298-7457, shaders/qwen38.metal:4761-5323 (rotary preparation, int8 append).
#include "q4_attention.h"
#include "q4_attention_plan.h"

#include <cuda_fp8.h>

#include <algorithm>

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

// Work of a thread: eight values, or the two eights of eight pairs, so that it owns both values of a pair and a call may work in place. Halves
// that do not begin at a multiple of eight values go by single pairs and values that are not turned.
constexpr uint32_t kRotaryThreads = 256;
__host__ __device__ inline bool by_eights(const RotaryView &r) { return r.interleaved || r.pairs % 8 == 0; }
__host__ __device__ inline uint32_t head_units(const RotaryView &r, uint32_t head_dim) {
    return !by_eights(r) ? head_dim - r.pairs : r.interleaved ? head_dim / 8 : (head_dim - r.pairs) / 8;
}

// A block turns `heads` heads of one token; the grid is [tokens][groups of heads]. Bound by memory. A thread has one unit, whose loads go out
// before the block's turns are computed. (2048 tokens of 24 x 256 values, 64 of them turned, fp32 in and bf16 out: a thread a pair 36 us;
// a block a token, whose threads take several units in turn, 21 us; this 15.8 us, 18.0 us with registers for five blocks an SM, 21 us for
// eight, which spill. 11.5 us at the peak. Halves that are not a multiple of eight values have a value a thread, whose loads and stores of two or
// four bytes are the bound: the same tokens with 36 to 130 values turned 71 to 75 us; interleaved pairs need no such form, 15 us.)
__global__ void __launch_bounds__(kRotaryThreads, 6) rotary_kernel(const RotaryParams p, uint32_t heads) {
    __shared__ float2 cs[kMaxHeadDim / 2];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t = blockIdx.x;
    const uint32_t first_head = blockIdx.y * heads, pairs = p.rotary.pairs, per_head = head_units(p.rotary, p.head_dim);
    const uint32_t h = threadIdx.x / per_head, c = threadIdx.x - h * per_head;
    const bool works = h < min(heads, p.heads - first_head), eights = by_eights(p.rotary);
    // first value of the unit, and whether it is the first of a pair's (or of eight pairs') with the others `pairs` behind it
    const bool both = eights ? !p.rotary.interleaved && c < pairs / 8 : c < pairs;
    const uint32_t d = (eights ? c * 8 : c) + (both || p.rotary.interleaved ? 0 : pairs);
    const uint64_t x = t * p.x_stride + (uint64_t)(first_head + h) * p.head_dim + d, o = t * p.out_stride + (uint64_t)(first_head + h) * p.head_dim + d;
    float a[8], b[8];
    if (works && eights) {
        load8(p.x, x, p.x_is_f32, a);
        if (both) load8(p.x, x + pairs, p.x_is_f32, b);
    } else if (works) {
        a[0] = load1(p.x, x, p.x_is_f32);
        if (both) b[0] = load1(p.x, x + pairs, p.x_is_f32);
    }
    const int32_t position = p.positions[t];
    for (uint32_t i = threadIdx.x; i < pairs; i += kRotaryThreads) cs[i] = turn(p.rotary, i, position);
    __syncthreads();
    if (!works) return;
    if (eights) {
        if (both) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 w = cs[d + j];
                const float va = a[j], vb = b[j];
                a[j] = va * w.x - vb * w.y;
                b[j] = vb * w.x + va * w.y;
            }
            store8(p.out, o + pairs, p.out_is_f32, b);
        }
        if (p.rotary.interleaved) turn_interleaved(a, d / 2, pairs, cs);
        store8(p.out, o, p.out_is_f32, a);
    } else if (both) {
        const float2 w = cs[d];
        store1(p.out, o, p.out_is_f32, a[0] * w.x - b[0] * w.y);
        store1(p.out, o + pairs, p.out_is_f32, b[0] * w.x + a[0] * w.y);
    } else {
        store1(p.out, o, p.out_is_f32, a[0]);
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
    uint64_t row, scale;  // of head 0: byte, and scale
    int32_t position, sequence;
    bool stands;  // not padded, not outside the cache
};

__device__ __forceinline__ int32_t sequence_of(const KvTokensParams &p, uint64_t t) { return p.sequences ? p.sequences[t] : (int32_t)(t / p.run); }

__device__ __forceinline__ Place place_of(const KvTokensParams &p, uint64_t t) {
    Place a;
    a.row = a.scale = 0;
    a.stands = false;
    a.position = p.positions[t];
    a.sequence = sequence_of(p, t);
    if (a.position < 0) return a;
    const uint32_t entry = (uint32_t)a.position / p.kv.page_tokens;
    if ((uint32_t)a.sequence < p.kv.sequences && entry < p.kv.per_sequence) {
        const uint32_t slot = (uint32_t)a.position - entry * p.kv.page_tokens;
        const uint32_t page = (uint32_t)p.kv.table[(uint64_t)a.sequence * p.kv.row_stride + entry];
        a.stands = page < p.kv.pages;
        a.row = (uint64_t)page * p.kv.page_stride + (uint64_t)slot * p.kv.token_stride;
        a.scale = (uint64_t)page * p.kv.kv_heads * p.kv.page_tokens + slot;
    }
    if (!a.stands) *p.kv.input_error = 1;
    return a;
}

// Rows of a block's tokens: keys and values of every head; a warp takes 32 / LANES rows at a time.
struct Row {
    uint32_t token, i;  // token of the block; head, or kv_heads + head for values
    __device__ __forceinline__ Row(uint32_t r, uint32_t a_token) : token(r / a_token), i(r % a_token) {}
    __device__ __forceinline__ void advance(Row by, uint32_t a_token) {
        token += by.token;
        i += by.i;
        if (i >= a_token) i -= a_token, ++token;
    }
};

// The eight values of a lane: two fours. Of fp32 rows they lie apart, so that what a warp asks for, or stores, at once has no gaps (4096 tokens of
// int8 written and read back 28 us with them side by side).
struct Fours {
    uint32_t a, b;
};
template <int LANES>
__device__ __forceinline__ Fours fours_of(uint32_t part, uint32_t e, bool apart) {
    const uint32_t a = apart ? (2 * e * LANES + part) * 4 : (e * LANES + part) * 8;
    return {a, a + (apart ? LANES * 4 : 4)};
}
__device__ __forceinline__ void load4(const void *base, uint64_t at, float *v) {
    const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
}

constexpr uint32_t kMostTokens = 8;  // of a block
constexpr uint32_t kRowsAhead = 4;   // eights of values that are on their way to a lane

// A block writes up to kMostTokens tokens. Of several tokens with the same place the last one is kept: every block looks through the tokens
// behind its own (most by one comparison with the range of its positions) while its first rows are on their way. A row is LANES lanes with
// EIGHTS eights of values each: two where keys are not turned (the other value of a pair is an eight of another lane), which halves what a
// row costs beside its values. Bound by instructions for long prompts, which keep the issue slots half busy, and by latency for single tokens.
// With the read kernel, for 4096 tokens of 2 x 4 x 256 fp32 values in int8: 25 us (84 MB, 12.8 us at the peak); with one eight a lane 2 us more;
// rows loaded behind the scan 36 us; registers for three blocks an SM 34 us; a block a token with whole warps for every row 54 us.
// Writing 4096 tokens of 2 x 4 x 256, us for fp32 / bf16 in: int8 16 / 20, with 64 values of a key turned 20 / 26, with all turned 26 / 30; e4m3
// 16 / 14, 20 / 21, 26 / 27; bf16 14 / 12, 17 / 17, 23 / 23. Looking through the tokens behind a block's own grows with the square of a call's: int8 from
// bf16 of 32768 / 65536 / 131072 / 262144 tokens of one sequence 122 / 274 / 743 / 2280 us, in 16 equal runs without sequence numbers, where a run ends
// the search, 114 / 217 / 431 / 878. (The quantising forms for fp32 rows spill 36 bytes at the 64 registers of four blocks an SM, others up to 8.)
template <int FMT, int LANES, int EIGHTS, bool TURN, bool F32>
__global__ void __launch_bounds__(256, 4) kv_write_kernel(const KvTokensParams p, uint32_t block_tokens) {
    __shared__ float2 cs[TURN ? kMostTokens : 1][kMaxHeadDim / 2];
    __shared__ Place places[kMostTokens];
    __shared__ uint32_t found[8];  // a bit a token: one behind it has the same place
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t0 = (uint64_t)blockIdx.x * block_tokens;
    const uint32_t tokens = (uint32_t)min((uint64_t)block_tokens, p.tokens - t0), pairs = p.rotary.pairs;
    constexpr uint32_t kAhead = kRowsAhead / EIGHTS;
    const uint32_t lane = threadIdx.x & 31u, part = lane % LANES, rows = tokens * 2 * p.kv.kv_heads;
    const uint32_t step = (blockDim.x >> 5) * (32 / LANES);
    const uint32_t kv_heads = p.kv.kv_heads;
    float v[kAhead][EIGHTS][8];  // fours_of(part, e)
    uint32_t r0 = (threadIdx.x >> 5) * (32 / LANES);
    const Row by(step, 2 * kv_heads);
    Row loads(r0 + lane / LANES, 2 * kv_heads), row = loads;
    const auto load_rows = [&]() {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k, loads.advance(by, 2 * kv_heads)) {
            const bool values = loads.i >= kv_heads;
            const void *in = values ? p.v_in : p.k_in;
            const bool has = loads.token < tokens && in;
            const uint64_t from = (t0 + loads.token) * (values ? p.v_stride : p.k_stride) + (loads.i - (values ? kv_heads : 0u)) * p.kv.head_dim;
#pragma unroll
            for (uint32_t e = 0; e < EIGHTS; ++e) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[k][e][j] = 0.f;
                const Fours at = fours_of<LANES>(part, e, F32);
                if (has && F32) {
                    if (at.a < p.kv.head_dim) load4(in, from + at.a, v[k][e]);
                    if (at.b < p.kv.head_dim) load4(in, from + at.b, v[k][e] + 4);
                } else if (has && at.a < p.kv.head_dim) {
                    load8(in, from + at.a, TURN ? p.is_f32 : 0u, v[k][e]);
                }
            }
        }
    };
    load_rows();
    if (threadIdx.x < tokens) places[threadIdx.x] = place_of(p, t0 + threadIdx.x);
    if (TURN)
        for (uint32_t i = threadIdx.x; i < tokens * pairs; i += blockDim.x) {
            const uint32_t t = i / pairs;
            cs[t][i - t * pairs] = turn(p.rotary, i - t * pairs, p.positions[t0 + t]);
        }
    // Tokens behind the block's first are looked through four at a time, from the first whose position starts at 16 bytes. Runs of one length
    // end the search with the last token's own.
    int32_t low = 0x7fffffff, high = -1;
#pragma unroll 1
    for (uint32_t t = 0; t < tokens; ++t) {
        const int32_t position = p.positions[t0 + t];
        if (position >= 0) low = min(low, position), high = max(high, position);
    }
    uint32_t replaced = 0;
    const uint64_t behind = t0 + 1, end = p.sequences ? p.tokens : min(p.tokens, (t0 + tokens - 1) / p.run * p.run + p.run);
    const uint64_t fours = min(end, behind + (0u - (uint32_t)((uintptr_t)(p.positions + behind) >> 2) & 3u)), last = fours + ((end - min(fours, end)) & ~3ull);
    const auto compare = [&](uint64_t u, int32_t position) {
        if (position < low || position > high) return;
        const int32_t sequence = sequence_of(p, u);
#pragma unroll 1
        for (uint32_t t = 0; t < tokens; ++t)
            if (position == p.positions[t0 + t] && sequence == sequence_of(p, t0 + t) && u > t0 + t) replaced |= 1u << t;
    };
    if (threadIdx.x < fours - min(behind, fours)) compare(behind + threadIdx.x, p.positions[behind + threadIdx.x]);
    if (threadIdx.x < end - last) compare(last + threadIdx.x, p.positions[last + threadIdx.x]);
#pragma unroll 2
    for (uint64_t u = fours + 4 * threadIdx.x; u < last; u += 4 * blockDim.x) {
        const int4 position = *reinterpret_cast<const int4 *>(p.positions + u);
        if (min(min(position.x, position.y), min(position.z, position.w)) > high || max(max(position.x, position.y), max(position.z, position.w)) < low) continue;
        const int32_t at[4] = {position.x, position.y, position.z, position.w};
        int32_t sequence[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sequence[i] = sequence_of(p, u + i);
#pragma unroll 1
        for (uint32_t t = 0; t < tokens; ++t) {
            const int32_t own = p.positions[t0 + t], own_sequence = sequence_of(p, t0 + t);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at[i] == own && sequence[i] == own_sequence && u + i > t0 + t) replaced |= 1u << t;
        }
    }
    replaced = __reduce_or_sync(0xffffffffu, replaced);
    if (lane == 0) found[threadIdx.x >> 5] = replaced;
    __syncthreads();
    replaced = __reduce_or_sync(0xffffffffu, lane < 8 ? found[lane] : 0u);
#pragma unroll 1
    for (;;) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k, row.advance(by, 2 * kv_heads)) {
            if (r0 + k * step >= rows) break;
            const bool values = row.i >= kv_heads;
            const uint32_t head = row.i - (values ? kv_heads : 0u), at = min(row.token, tokens - 1);
            const bool writes = row.token < tokens && (values ? p.v_in : p.k_in) && places[at].stands && !(replaced >> at & 1u);
            if (TURN) {
                const uint32_t d = part * 8;
                const bool turns = !values && d < 2 * pairs;
                if (p.rotary.interleaved) {
                    if (turns) turn_interleaved(v[k][0], d / 2, pairs, cs[at]);
                } else if (pairs % 8 == 0) {
                    // the other values of the pairs are those of a lane of the same row
                    const uint32_t by = pairs / 8, other = (lane & ~(LANES - 1u)) + (part < by ? part + by : part - by) % LANES;
                    const uint32_t i = part < by ? d : d - pairs;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float b = __shfl_sync(0xffffffffu, v[k][0][j], other);
                        if (turns) v[k][0][j] = v[k][0][j] * cs[at][i + j].x + (part < by ? -b : b) * cs[at][i + j].y;
                    }
                } else if (turns && writes) {
                    const uint64_t key = (t0 + at) * p.k_stride + head * p.kv.head_dim;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t e = d + j;
                        if (e < pairs) v[k][0][j] = v[k][0][j] * cs[at][e].x - load1(p.k_in, key + e + pairs, p.is_f32) * cs[at][e].y;
                        else if (e < 2 * pairs) v[k][0][j] = v[k][0][j] * cs[at][e - pairs].x + load1(p.k_in, key + e - pairs, p.is_f32) * cs[at][e - pairs].y;
                    }
                }
            }
            uint8_t *const to = (values ? p.kv.v : p.kv.k) + places[at].row + head * p.kv.head_stride;
            if (FMT == 0) {
#pragma unroll
                for (uint32_t e = 0; e < EIGHTS; ++e) {
                    const Fours to_of = fours_of<LANES>(part, e, F32);
                    const uint4 w = pack8_bf16(v[k][e]);
                    if (!F32) {
                        if (writes && to_of.a < p.kv.head_dim) *reinterpret_cast<uint4 *>(to + to_of.a * 2) = w;
                        continue;
                    }
                    if (writes && to_of.a < p.kv.head_dim) *reinterpret_cast<uint2 *>(to + to_of.a * 2) = make_uint2(w.x, w.y);
                    if (writes && to_of.b < p.kv.head_dim) *reinterpret_cast<uint2 *>(to + to_of.b * 2) = make_uint2(w.z, w.w);
                }
                continue;
            }
            uint32_t amax = 0;
#pragma unroll
            for (uint32_t e = 0; e < EIGHTS; ++e)
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[k][e][j]) & 0x7fffffffu);
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
            const bool finite = amax < 0x7f800000u;
            const float scale = finite ? __fdiv_rn(__uint_as_float(amax), FMT == 1 ? 127.f : 448.f) : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (uint32_t e = 0; e < EIGHTS; ++e) {
                const Fours to_of = fours_of<LANES>(part, e, F32);
                if (!writes || to_of.a >= p.kv.head_dim) continue;
                const uint2 w = finite ? encode8<FMT == 0 ? 1 : FMT>(v[k][e], scale) : make_uint2(0u, 0u);
                if (!F32) {
                    *reinterpret_cast<uint2 *>(to + to_of.a) = w;
                    continue;
                }
                *reinterpret_cast<uint32_t *>(to + to_of.a) = w.x;
                if (to_of.b < p.kv.head_dim) *reinterpret_cast<uint32_t *>(to + to_of.b) = w.y;
            }
            if (writes && part == 0) (values ? p.kv.v_scales : p.kv.k_scales)[kv_scale_index(places[at].scale, head, p.kv.page_tokens)] = scale;
        }
        r0 += kAhead * step;
        if (r0 >= rows) break;
        load_rows();
    }
}

// The reverse, number = code * scale rounded to the output's type. Bound by memory for long prompts (4096 int8 tokens of 2 x 4 x 256 values to fp32,
// 42 MB: 10 us, 6.4 at the peak), else by the latencies of position, page number and row, which depend on one another.
template <int FMT, int LANES, bool F32>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvTokensParams p, uint32_t block_tokens) {
    __shared__ Place places[kMostTokens];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t0 = (uint64_t)blockIdx.x * block_tokens;
    const uint32_t tokens = (uint32_t)min((uint64_t)block_tokens, p.tokens - t0);
    if (threadIdx.x < tokens) places[threadIdx.x] = place_of(p, t0 + threadIdx.x);
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31u, step = (blockDim.x >> 5) * (32 / LANES);
    const Fours d = fours_of<LANES>(lane % LANES, 0, F32);
    const bool second = !F32 || d.b < p.kv.head_dim;
    if (d.a >= p.kv.head_dim) return;
    const uint32_t kv_heads = p.kv.kv_heads;
    const Row by(step, 2 * kv_heads);
    Row loads((threadIdx.x >> 5) * (32 / LANES) + lane / LANES, 2 * kv_heads), row = loads;
#pragma unroll 1
    while (row.token < tokens) {
        uint4 held[kRowsAhead];
        float scale[kRowsAhead];
        bool there[kRowsAhead];
#pragma unroll
        for (uint32_t k = 0; k < kRowsAhead; ++k, loads.advance(by, 2 * kv_heads)) {
            const bool values = loads.i >= kv_heads;
            const uint32_t head = loads.i - (values ? kv_heads : 0u);
            there[k] = loads.token < tokens && (values ? p.v_out : p.k_out) && places[loads.token].stands;
            held[k] = make_uint4(0u, 0u, 0u, 0u);
            scale[k] = 1.f;
            if (!there[k]) continue;
            const uint8_t *from = (values ? p.kv.v : p.kv.k) + places[loads.token].row + head * p.kv.head_stride;
            if (FMT == 0) {
                if (!F32) {
                    held[k] = *reinterpret_cast<const uint4 *>(from + 2 * d.a);
                    continue;
                }
                const uint2 a = *reinterpret_cast<const uint2 *>(from + 2 * d.a), b = second ? *reinterpret_cast<const uint2 *>(from + 2 * d.b) : make_uint2(0u, 0u);
                held[k] = make_uint4(a.x, a.y, b.x, b.y);
            } else {
                if (!F32) {
                    const uint2 c = *reinterpret_cast<const uint2 *>(from + d.a);
                    held[k].x = c.x, held[k].y = c.y;
                } else {
                    held[k].x = *reinterpret_cast<const uint32_t *>(from + d.a);
                    if (second) held[k].y = *reinterpret_cast<const uint32_t *>(from + d.b);
                }
                scale[k] = (values ? p.kv.v_scales : p.kv.k_scales)[kv_scale_index(places[loads.token].scale, head, p.kv.page_tokens)];
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kRowsAhead; ++k, row.advance(by, 2 * kv_heads)) {
            if (!there[k]) continue;
            const bool values = row.i >= kv_heads;
            float v[8];
            if (FMT == 0) unpack8_bf16(held[k], v);
            else decode8<FMT == 0 ? 1 : FMT>(make_uint2(held[k].x, held[k].y), scale[k], v);
            const uint64_t to = (t0 + row.token) * (values ? p.v_stride : p.k_stride) + (row.i - (values ? kv_heads : 0u)) * p.kv.head_dim;
            if (F32) {
                float *const out = static_cast<float *>(values ? p.v_out : p.k_out) + to;
                *reinterpret_cast<float4 *>(out + d.a) = make_float4(v[0], v[1], v[2], v[3]);
                if (second) *reinterpret_cast<float4 *>(out + d.b) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                store8(values ? p.v_out : p.k_out, to + d.a, 0, v);
            }
        }
    }
}

// Tokens of a block: few tokens go to as many blocks as there are, many in eights. (4096 tokens: four a block 30 us, seven 35 us.)
uint32_t block_tokens(uint64_t tokens, uint32_t sm_count) { return (uint32_t)(tokens / (8ull * sm_count) < kMostTokens ? tokens / (8ull * sm_count) + 1 : kMostTokens); }

template <int FMT, int LANES>
cudaError_t launch_tokens(const KvTokensParams &p, bool write, uint32_t sm_count, cudaStream_t stream) {
    const uint32_t each = block_tokens(p.tokens, sm_count);
    const auto kernel = !write                     ? (p.is_f32 ? kv_read_kernel<FMT, LANES, true> : kv_read_kernel<FMT, LANES, false>)
                        : p.rotary.step && p.k_in ? kv_write_kernel<FMT, LANES, 1, true, false>
                        : p.is_f32                ? kv_write_kernel<FMT, LANES / 2, 2, false, true>
                                                  : kv_write_kernel<FMT, LANES / 2, 2, false, false>;
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
    // heads of a block: a unit a thread, or fewer where there are few tokens
    const uint32_t most = q4::kRotaryThreads / q4::head_units(p->rotary, p->head_dim);
    const uint64_t groups = std::max<uint64_t>(2ull * sm_count / p->tokens, 1);
    const uint32_t heads = (uint32_t)std::min<uint64_t>(most, (p->heads + groups - 1) / groups);
    return q4::launch_dependent(q4::rotary_kernel, dim3((uint32_t)p->tokens, (p->heads + heads - 1) / heads), q4::kRotaryThreads, 0, stream, *p, heads);
}

extern "C" cudaError_t q4k_kv_write(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream) {
    return q4::launch_tokens(*p, true, sm_count, stream);
}

extern "C" cudaError_t q4k_kv_read(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream) {
    return q4::launch_tokens(*p, false, sm_count, stream);
}
