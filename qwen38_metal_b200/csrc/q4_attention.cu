// Attention of new tokens over a paged cache. Counterparts in the reference: the cache's scores and values kernels
// (src/metal_runtime.rs:8230-8798, shaders/qwen38.metal:4761-5323).
//
//     out = sum_j p_j v_j / sum_j p_j,   p_j = e^(scale q.k_j)
//
// Every key and value is read once from memory for 8, 16 or 24 query rows (token, head) that share its key head: at one byte a value and 8 rows
// that is 12 to 16 operations a byte, so memory is the bound, and the kernel is built around keeping loads in flight.
//
//   * One block per SM: eight warps that multiply and one that asks for tiles with tensor copies into a ring in shared memory, keys of
//     128 tokens (256 where rows are short) and their values in turn, past the end of an item too: 190 KB are in flight while results
//     are written. A page has a whole number of the 16-token rows that a copy brings; copies of single segments of rows, and scales as
//     copies of their own, were more than the copy engine takes (1100 of 4300 cycles for 128 tokens).
//   * Warp w has the scores of an eighth of the tile's tokens, hands their weights on through shared memory, and then adds up an eighth of
//     the dimensions of the values for all of them: one barrier for a tile, and a result lies in few registers. (Warps that kept whole
//     results of tokens of their own needed 128 registers for them and four rounds through shared memory to join them: 3 us for every
//     item, 8 for a cut one. Two groups of four warps that took turns at tiles were no faster on long contexts and slower on others.)
//   * Both products run on MMAs with eight query rows: rows 0...7 of the left operand hold the upper halves of the eight rows' factors,
//     rows 8...15 the lower halves, so that the sum of the two accumulators is a product of factors of 16 bits or more (two bf16
//     numbers, error 2^-17; two fp16 numbers for 8-bit caches, 2^-22), at no cost: the rows would be empty.
//   * int8 codes are multiplied as they lie in memory, by whole-number MMAs with four 8-bit digits of every query, and of every weight.
//     e4m3 codes become fp16 exactly. Which dimensions (or tokens) an MMA multiplies is free as long as its operands agree, so that a
//     lane takes whole 16-byte pieces of a key row; values are read transposed as pairs of bytes, which gives the lane a pair of
//     dimensions, one for each of two MMAs, and a byte permutation for each brings four tokens into a register.
//   * One pass: sums and results are relative to a power of two for each row that is raised when a score lies 8 above it, which is seldom
//     after the first tiles. The scale of a token's values goes into its weight; weights times scales are lifted by a power of two of their
//     own, so that they stay in range whatever the scales are, and whatever values lie behind a score that jumps.
//   * The work of all sequences is cut into equal shares by every block for itself (q4_attention_plan.h), from the lengths in device memory:
//     a captured graph follows them. Results of an item cut over several blocks are joined in order by the last one.
//
// Measured, 24 query heads on 4 key heads of 256: one sequence of 262144 int8 tokens 93 to 99 us (545 MB, 5.5 to 5.8 TB/s), of 8200 tokens 13.2 us, 32
// sequences of 500 to 8000 tokens 58 to 61 us (277 MB); four sequences of 9001 to 20011 bf16 tokens with four new ones each 53 us (214 MB, 35 us of it in
// the loop at 6.1 TB/s, the rest is start and joining; 2.8e-6 from 64 bits, 1.8e-6 of it by the weights' two halves; sums in 32 bits 2.1e-6); 32 heads on 8 of 128, 128 sequences of 3100 to 5100 e4m3 tokens 221 to 227 us (1.11 GB, 5.0 TB/s).
#include <cuda_fp8.h>

#include <atomic>

#include "q4_attention.h"
#include "q4_attention_plan.h"
#include "q4_device.cuh"
#include "q4_tensor_map.h"

namespace q4 {

constexpr uint32_t kWarps = 8, kMultipliers = kWarps * 32, kThreads = kMultipliers + 32, kAllWarps = kWarps + 1;  // the last warp asks for tiles
constexpr uint32_t kMostBlocks = 256;           // of a launch
constexpr uint32_t kMostSets = 3;               // of eight query rows that a block takes through a tile together
constexpr uint32_t kLeastRun = 16;              // tiles: shorter runs cost more in joining than they save
constexpr float kNone = -3.0e38f;               // a reference below all scores: the row has seen nothing
constexpr float kHeadroom = 8.f;                // how far above its reference a score may lie, in powers of two
constexpr float kMostLift = 126.f;              // of weights times scales, in powers of two: its reciprocal is a number of 32 bits
// 8-bit caches: the largest weight times scale is brought below 2^11 (int8: 2^26) when the lift is set and may grow to 2^15 (2^30). As fp16
// halves, up to the end of fp16's range, weights keep 16 bits down to 2^-19 of the largest one (and 2^-35 of it below); as whole
// numbers they are off by half at most, 2^-26 of the largest one. The factor that brings them there is 2^126 at most, whose reciprocal 32 bits
// hold: largest ones below 2^-100 (int8) keep fewer bits.
template <int FMT>
struct Weights {
    static constexpr int kExponent = FMT == 1 ? 26 : 11;
    static constexpr float kMost = FMT == 1 ? 1073741824.f : 32768.f;
};
constexpr unsigned long long kWaitLimitNs = 200ull * 1000 * 1000, kLateLimitNs = 1000 * 1000;
constexpr uint32_t kSharedLimit = 227 * 1024;

template <int FMT, int HDP, int SETS>
struct Shape {
    static constexpr uint32_t kRows = SETS * kAttentionRows;         // query rows of an item
    static constexpr uint32_t kRow = HDP * (FMT == 0 ? 2 : 1);       // bytes of a token's row in shared memory
    static constexpr uint32_t kSeg = kRow < 128 ? kRow : 128;        // swizzled together
    static constexpr uint32_t kSegs = kRow / kSeg;
    static constexpr uint32_t kSub = kTileTokens * kRow;             // 16 tokens' keys or values
    static constexpr uint32_t kOwnSubs = kRow > 256 ? 1 : 2;         // of a tile, whose scores a warp has
    static constexpr uint32_t kSubs = kWarps * kOwnSubs;             // of a tile
    static constexpr uint32_t kSlot = kSubs * kSub;                  // of the ring: keys, or values, of a tile
    static constexpr uint32_t kPieces = kSeg / 64;                   // 16-byte pieces of a segment a lane takes from a key row
    static constexpr uint32_t kWords = FMT == 2 ? 8 : 4;             // registers of a 16-byte piece as it is multiplied
    static constexpr uint32_t kMmas = HDP / 16;                      // per 8 tokens of scores
    static constexpr uint32_t kChunkDims = FMT == 0 ? 8 : 16;        // of a 16-byte piece
    static constexpr uint32_t kValueWarps = HDP / kChunkDims < kWarps ? HDP / kChunkDims : kWarps;  // that have dimensions of the values
    static constexpr uint32_t kWarpDims = HDP / kValueWarps;
    static constexpr uint32_t kChunks = kWarpDims / kChunkDims;
    static constexpr uint32_t kAcc = kWarpDims / 8;                  // accumulators of four numbers
    static constexpr uint32_t kOwn = kWarpDims / 4;                  // numbers of a row's result in a lane
    static constexpr bool kQueriesStay = HDP < 256 && SETS == 1;  // in registers
    static constexpr uint32_t kTogether = SETS < 3 ? 2 * kOwnSubs : 2;   // eights of tokens whose scores are computed together
    // shared memory: ring, scales of its keys and values, weights, queries, barriers, small arrays
    static constexpr uint32_t kScales = FMT == 0 ? 0 : 2 * kSubs * 64;  // of a slot
    static constexpr uint32_t kSetQueries = kMmas * 32 * 16, kQueries = SETS * kSetQueries;
    static constexpr uint32_t kSetWeights = kSubs * 32 * 16, kWeights = SETS * kSetWeights;  // of a tile; there are two
    static constexpr uint32_t kSmall = (3 * kWarps + 1) * kRows * 4 + 3 * kAllWarps * 4 + 12 * 4;
    static constexpr uint32_t kFit = (kSharedLimit - 1024 - kQueries - 2 * kWeights - kSmall) / (kSlot + kScales + 16);
    static constexpr uint32_t kSlots = kFit < 16 ? kFit : 16;
    static constexpr uint32_t kShared = 1024 + kSlots * (kSlot + kScales + 16) + kQueries + 2 * kWeights + kSmall;
    static_assert(kSlots >= 2 && kSubs * kSegs <= 32 && 2 * kWeights >= kMostBlocks * kRows * 4 && kSmall % 4 == 0 && kShared <= kSharedLimit, "");
};

// ---- small pieces ----

__device__ __forceinline__ float exp2_fast(float x) {  // 2 units in the last place; below 2^-126: zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}

// Two numbers as upper and lower halves: a = hi + lo up to 2^-17 (bf16) or 2^-22 (fp16, numbers up to 2).
template <int FMT>
__device__ __forceinline__ void split(float a, float b, uint32_t &hi, uint32_t &lo) {
    if (FMT == 0) {
        hi = pack_bf16(a, b);
        lo = pack_bf16(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
    } else {
        hi = pack_f16(a, b);
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
        lo = pack_f16(a - f.x, b - f.y);
    }
}

template <int FMT>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (FMT == 0)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        mma_f16_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}

// Queries against int8 codes: whole-number MMAs of four signed 8-bit digits of each query, two digits to a call.
__device__ __forceinline__ void split_digits(const float (&q)[8], uint4 &upper, uint4 &lower) {
    uint32_t word[4][2] = {{0u, 0u}, {0u, 0u}, {0u, 0u}, {0u, 0u}};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        int v = __float2int_rn(q[i] * 0x1p29f);  // |q| < 2
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int digit = k == 3 ? v : (int)(int8_t)(v & 0xff);
            word[k][i / 4] |= ((uint32_t)digit & 0xffu) << (i % 4 * 8);
            v = (v - digit) >> 8;
        }
    }
    upper = make_uint4(word[3][0], word[2][0], word[3][1], word[2][1]);
    lower = make_uint4(word[1][0], word[0][0], word[1][1], word[0][1]);
}

// A number from the sums of products with its factor's four digits. Sums of up to 256 products of 8-bit numbers are at most 2^22, which
// small_int_to_float takes; the conversion unit (8 cycles an instruction) would be busy for a fifth of the time.
__device__ __forceinline__ float of_digits(int d3, int d2, int d1, int d0) {
    return fmaf(fmaf(small_int_to_float(d3), 256.f, small_int_to_float(d2)), 65536.f, fmaf(small_int_to_float(d1), 256.f, small_int_to_float(d0)));
}

// The four signed digits of four whole numbers 0 ... 2^30, a word for each digit from the highest on. With 128 added to its lower three
// digits, a number's bytes are its digits, each but the highest plus 128.
__device__ __forceinline__ void weight_digits(const float (&w)[4], uint32_t (&digit)[4]) {
    uint32_t n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = (uint32_t)__float2int_rn(w[i]) + 0x00808080u;
    const uint32_t low01 = __byte_perm(n[0], n[1], 0x5140), low23 = __byte_perm(n[2], n[3], 0x5140);    // bytes 0, 0, 1, 1
    const uint32_t high01 = __byte_perm(n[0], n[1], 0x7362), high23 = __byte_perm(n[2], n[3], 0x7362);  // bytes 2, 2, 3, 3
    digit[3] = __byte_perm(low01, low23, 0x5410) ^ 0x80808080u;
    digit[2] = __byte_perm(low01, low23, 0x7632) ^ 0x80808080u;
    digit[1] = __byte_perm(high01, high23, 0x5410) ^ 0x80808080u;
    digit[0] = __byte_perm(high01, high23, 0x7632);
}
// Four e4m3 numbers as fp16, exactly.
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t &lower, uint32_t &upper) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lower), "=r"(upper) : "r"(w));
}

__device__ __forceinline__ void ldmatrix_x2_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded: after the limit the call is reported as failed and goes on with what is there, with a shorter limit for what follows.
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, unsigned long long &limit, int *error_flag) {
    if (mbar_try(bar, parity)) return;
    unsigned long long begin = 0;
    for (uint32_t spin = 1; spin != 0; ++spin) {
        if (mbar_try(bar, parity)) return;
        if ((spin & 255u) == 0) {
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (begin == 0) begin = now;
            if (now - begin > limit) break;
        }
    }
    limit = kLateLimitNs;
    *error_flag = 1;
}

// Barrier of the warps that multiply; the second one tells whether any thread brought `true`.
__device__ __forceinline__ void multipliers_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kMultipliers) : "memory"); }
__device__ __forceinline__ bool multipliers_any(bool mine) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((uint32_t)mine), "n"(kMultipliers) : "memory");
    return any != 0;
}

__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int token, int head, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(token),
                 "r"(head), "r"(page)
                 : "memory");
}
__device__ __forceinline__ void copy_whole_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int token, int head, int page) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(token),
                 "r"(head), "r"(page)
                 : "memory");
}
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 16 bytes, or zeros; counted by a barrier when they and the thread's others have arrived
__device__ __forceinline__ void copy_16_or_zeros(uint32_t dst, const void *src, bool wanted) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(wanted ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

// ---- a block's share ----

struct Geometry {
    uint32_t chunks;  // items of a key head: 8, 16 or 24 query rows each
    uint32_t heads;   // items of a sequence = key heads * chunks
    uint32_t rows;    // query rows of a key head
    uint32_t group;   // query heads of a key head
    uint32_t whole_rows;  // a copy brings all segments of 16 rows, else one of them
    uint32_t tile_shift;  // a copy brings 16 << tile_shift tokens (rows of one segment)
    AttentionPages pages;
};

__device__ __forceinline__ int64_t length_of(const AttentionParams &p, uint32_t s) {
    const int64_t n = __ldcg(p.lengths + s), most = (int64_t)p.kv.per_sequence * p.kv.page_tokens;
    return n < 0 ? 0 : n > most ? most : n;
}

using Cursor = AttentionCursor;

struct Share {
    bool any;
    Cursor at;
    AttentionCut cut;
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= (uint32_t)off) v += o;
    }
    return v;
}

// All threads. `scratch`: 3 * kAllWarps words in shared memory. Up to 32 sequences every warp finds it by itself.
__device__ __forceinline__ Share share_of_block(const AttentionParams &p, const Geometry &g, uint32_t *scratch) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, sequences = p.kv.sequences;
    const bool few = sequences <= 32;
    const uint32_t mine = few ? lane : threadIdx.x, stride = few ? 32 : kThreads;
    const int64_t most = (int64_t)p.kv.per_sequence * p.kv.page_tokens;
    uint32_t tiles = 0, items = 0, longest = 0, own = 0;  // own: tiles of the thread's first sequence
#pragma unroll 1
    for (uint32_t s = mine; s < sequences; s += stride) {
        const int32_t raw = __ldcg(p.lengths + s);
        const uint32_t t = attention_tiles(raw > most ? most : raw, g.tile_shift);
        if ((raw < 0 || raw > most) && blockIdx.x == 0) *p.kv.input_error = 1;
        if (s == mine) own = t;
        tiles += t;
        items += t > 0;
        longest = max(longest, t);
    }
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    items = __reduce_add_sync(0xffffffffu, items);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (!few) {
        if (lane == 0) scratch[warp] = tiles, scratch[kAllWarps + warp] = items, scratch[2 * kAllWarps + warp] = longest;
        __syncthreads();
        const bool has = lane < kAllWarps;
        tiles = __reduce_add_sync(0xffffffffu, has ? scratch[lane] : 0u);
        items = __reduce_add_sync(0xffffffffu, has ? scratch[kAllWarps + lane] : 0u);
        longest = __reduce_max_sync(0xffffffffu, has ? scratch[2 * kAllWarps + lane] : 0u);
    }
    Share share;
    share.any = false;
    share.at = Cursor{};
    if (tiles == 0) return share;
    share.cut = attention_cut(tiles * g.heads, items * g.heads, longest, gridDim.x, kLeastRun >> g.tile_shift, g.tile_shift);
    uint32_t target;
    if (!attention_target(share.cut, blockIdx.x, &target)) return share;
    // the sequence that holds piece or tile number `target`; every warp finds it: first eight that do, of 256 at a time, then which of them
    uint32_t base = 0, before = 0, hit = 0, s = 0, start = 0;
    if (!few) {
#pragma unroll 1
        for (;; base += 256) {
            uint32_t weight = 0;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                const uint32_t i = base + lane * 8 + j;
                weight += attention_weight(share.cut, i < sequences ? attention_tiles(length_of(p, i), g.tile_shift) : 0u, g.heads);
            }
            const uint32_t to = before + warp_scan(weight, lane);
            hit = __ballot_sync(0xffffffffu, target >= to - weight && target - (to - weight) < weight);
            const uint32_t from = hit ? __ffs(hit) - 1 : 31;
            before = __shfl_sync(0xffffffffu, hit ? to - weight : to, from);
            if (hit) {
                base += from * 8;
                break;
            }
            if (sequences - base <= 256) return share;
        }
    }
    {
        const uint32_t i = base + lane, t = few ? own : lane < 8 && i < sequences ? attention_tiles(length_of(p, i), g.tile_shift) : 0u;
        const uint32_t weight = attention_weight(share.cut, t, g.heads), to = before + warp_scan(weight, lane);
        hit = __ballot_sync(0xffffffffu, target >= to - weight && target - (to - weight) < weight);
        const uint32_t from = hit ? __ffs(hit) - 1 : 0;
        s = base + from;
        start = __shfl_sync(0xffffffffu, to - weight, from);
    }
    if (hit) share.any = share.at.start(share.cut, target, s, start, [&](uint32_t i) { return length_of(p, i); }, sequences, g.heads);
    return share;
}

template <int FMT>
__device__ __forceinline__ bool not_finite(uint32_t w, uint32_t byte) {  // the value that begins at this byte of a word
    if (FMT == 0) return ((w >> (byte * 8)) & 0x7f80u) == 0x7f80u;
    return ((w >> (byte * 8)) & 0x7fu) == 0x7fu;
}

// A slot of the ring and the phase of its barriers.
template <uint32_t N>
struct Turn {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void next() {
        slot = slot + 1 == N ? 0 : slot + 1;
        phase ^= slot == 0;
    }
};

// ---- the warp that asks for tiles ----

// A lane brings a tile, or one segment of it where rows are not a whole number of segments; scales come in 16-byte pieces, two a lane.
// Page numbers are read while the slot that comes next is still in use.
template <int FMT, int HDP, int SETS>
__device__ __forceinline__ void ask_for_tiles(const AttentionParams &p, const Geometry &g, Cursor at, const CUtensorMap *k_map, const CUtensorMap *v_map, uint32_t ring, uint32_t scales,
                                              uint32_t full, uint32_t empty, uint32_t lane) {
    using S = Shape<FMT, HDP, SETS>;
    const uint32_t per = g.whole_rows ? 1 : S::kSegs, mine = lane / per, seg = lane % per;
    const auto lengths = [&](uint32_t i) { return length_of(p, i); };
    unsigned long long limit_ns = kWaitLimitNs;
    Turn<S::kSlots> turn;
    do {
        const uint32_t head = at.item / g.chunks;
        const int32_t *const table = p.kv.table + (uint64_t)at.s * p.kv.row_stride;
        const uint32_t shift = S::kSegs == 1 ? g.tile_shift : 0, tiles = S::kSubs >> shift;  // of a slot
        uint32_t entry = g.pages.page_of(at.begin + mine);
        uint32_t page = at.begin + mine < at.end ? (uint32_t)__ldcg(table + entry) : 0u;
        for (uint32_t tile = at.begin; tile < at.end; tile += tiles) {
            const uint32_t count = min(at.end - tile, tiles);
            const bool wanted = mine < count, there = page < p.kv.pages;
            // (a page outside the cache is outside the tensor map too: such copies bring zeros)
            const uint32_t now = there ? page : p.kv.pages, place = (tile + mine - entry * g.pages.per) * (kTileTokens << shift);
            if (wanted && !there) *p.kv.input_error = 1;
            const uint32_t next = tile + tiles + mine;
            if (next < at.end) {
                entry = g.pages.page_of(next);
                page = (uint32_t)__ldcg(table + entry);
            }
#pragma unroll
            for (uint32_t values = 0; values < 2; ++values) {
                mbar_wait(empty + turn.slot * 8, turn.phase ^ 1u, limit_ns, p.error_flag);
                const uint32_t bar = full + turn.slot * 8, dst = ring + turn.slot * S::kSlot;
                if (lane == 0) mbar_expect(bar, count * (S::kSub << shift));
                __syncwarp();
                if (wanted) {
                    if (S::kSegs > 1 && g.whole_rows) copy_whole_tile(dst + lane * S::kSub, values ? v_map : k_map, bar, (int)place, (int)head, (int)now);
                    else copy_tile(dst + lane * (kTileTokens * S::kSeg << shift), values ? v_map : k_map, bar, (int)(seg * S::kSeg / (FMT == 0 ? 2 : 1)), (int)place, (int)head, (int)now);
                }
                if (FMT != 0 && values == 0) {
                    // lane 4 i + j: 16-byte piece j of the scales of 16 tokens, of keys and of values
#pragma unroll
                    for (uint32_t of = lane / 4; of < S::kSubs; of += 8) {
                        const uint32_t by = (of >> shift) * per, of_page = __shfl_sync(0xffffffffu, now, by);
                        const uint32_t of_place = __shfl_sync(0xffffffffu, place, by) + (of & ((1u << shift) - 1)) * kTileTokens;
                        const bool here = of >> shift < count && of_page < p.kv.pages;
                        const uint64_t from = here ? ((uint64_t)of_page * p.kv.kv_heads + head) * p.kv.page_tokens + of_place + lane % 4 * 4 : 0;
                        const uint32_t sc = scales + turn.slot * S::kScales + of * 64 + lane % 4 * 16;
                        copy_16_or_zeros(sc, p.kv.k_scales + from, here);
                        copy_16_or_zeros(sc + S::kSubs * 64, p.kv.v_scales + from, here);
                    }
                }
                if (FMT != 0) copies_arrive(bar);
                turn.next();
            }
        }
    } while (at.next(lengths, p.kv.sequences, g.heads));
    if (FMT != 0) asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- the kernel ----

template <int FMT, int HDP, int SETS>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ Geometry g, const __grid_constant__ CUtensorMap k_map,
                                                                const __grid_constant__ CUtensorMap v_map) {
    using S = Shape<FMT, HDP, SETS>;
    extern __shared__ uint8_t shared_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(shared_raw), pad = (1024u - (raw & 1023u)) & 1023u;
    const uint32_t ring = raw + pad, scales = ring + S::kSlots * S::kSlot, weights = scales + S::kSlots * S::kScales, queries = weights + 2 * S::kWeights,
                   full = queries + S::kQueries, empty = full + S::kSlots * 8, joined = empty + S::kSlots * 8;
    float *const small = reinterpret_cast<float *>(shared_raw + (joined + 16 - raw));
    float *const highs = small, *const weight_highs = small + kWarps * S::kRows, *const sums = small + 2 * kWarps * S::kRows;  // [warp][row]
    float *const row_scales = small + 3 * kWarps * S::kRows;                                                                         // [row] scale of the scores, in powers of two
    uint32_t *const scratch = reinterpret_cast<uint32_t *>(row_scales + S::kRows), *const joins = scratch + 3 * kAllWarps;  // joins: 2 of 6 words
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, row = lane >> 2, quad = lane & 3u;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < S::kSlots; ++i) {
            mbar_init(full + i * 8, FMT != 0 ? 33 : 1);  // the tile copies; the lanes' scales
            mbar_init(empty + i * 8, kWarps);
        }
        mbar_init(joined, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    grid_dependency_wait();
    grid_dependents_launch();

    const Share share = share_of_block(p, g, scratch);
    const auto lengths = [&](uint32_t i) { return length_of(p, i); };
    if (share.any && warp == kWarps) {
        ask_for_tiles<FMT, HDP, SETS>(p, g, share.at, &k_map, &v_map, ring, scales, full, empty, lane);
    } else if (share.any) {
        Turn<S::kSlots> turn;
        unsigned long long limit_ns = kWaitLimitNs;
        uint32_t weights_at = weights;  // one of two
        Cursor at = share.at;
        // eight values of query row `warp` of each set of eight, as they lie in memory; those of the next item are on their way meanwhile where registers allow
        constexpr bool kAhead = SETS == 1;
        uint4 rows_in[SETS][2];
        const auto load_query = [&](const Cursor &c) {
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) {
                const uint32_t r = c.item % g.chunks * S::kRows + set * kAttentionRows + warp, d = lane * 8;
                rows_in[set][0] = rows_in[set][1] = make_uint4(0u, 0u, 0u, 0u);
                if (r < g.rows && d < p.kv.head_dim) {
                    const uint64_t base = ((uint64_t)c.s * p.q_tokens + r / g.group) * p.q_stride + ((uint64_t)(c.item / g.chunks) * g.group + r % g.group) * p.kv.head_dim + d;
                    const uint4 *const from = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p.q) + base * (p.q_is_f32 ? 4 : 2));
                    rows_in[set][0] = __ldcg(from);
                    if (p.q_is_f32) rows_in[set][1] = __ldcg(from + 1);
                }
            }
        };
        if (kAhead) load_query(at);
        constexpr uint32_t kPart = S::kRows * (kMaxHeadDim + 2);  // numbers of a partial result: rows, then maxima, then sums
        uint32_t left_parts = 0;  // partial results this block has left: two at most
        bool more;
        do {
            // ---- queries of the item: warp w splits row w into halves, or digits, in the order in which key rows are read ----
            const uint32_t head = at.item / g.chunks, chunk = at.item % g.chunks;
            if (!kAhead) load_query(at);
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) {
                const uint32_t d = lane * 8, w[8] = {rows_in[set][0].x, rows_in[set][0].y, rows_in[set][0].z, rows_in[set][0].w, rows_in[set][1].x, rows_in[set][1].y, rows_in[set][1].z, rows_in[set][1].w};
                float q[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = __uint_as_float(p.q_is_f32 ? w[i] : i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xffff0000u);
                float unit = 1.f, row_scale = p.scale * 1.4426950408889634f;
                if (FMT != 0) {
                    // fp16 halves, whole numbers: the row is scaled by a power of two that brings its largest value into [1, 2)
                    uint32_t amax = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(q[i]) & 0x7fffffffu);
                    amax = __reduce_max_sync(0xffffffffu, amax);
                    const uint32_t e = min(max(amax >> 23, 1u), 254u);
                    unit = e == 254u ? __uint_as_float(0x00400000u) : __uint_as_float((254u - e) << 23);
                    row_scale *= __uint_as_float(e << 23);
                    if (FMT == 1) row_scale *= 0x1p-29f;
                    if (amax >= 0x7f800000u) row_scale = __uint_as_float(0x7fc00000u);  // whole numbers hold no NaN
                }
                if (d < HDP) {
                    // a lane's part of an MMA is four values, of a whole-number one eight; a 16-byte piece of a key row holds 8 or 16
                    constexpr uint32_t kPer = S::kChunkDims / 4;
                    const uint32_t piece = d / S::kChunkDims, seg = piece / (S::kSeg / 16), in_seg = piece % (S::kSeg / 16);
                    const uint32_t m = (seg * S::kPieces + in_seg % S::kPieces) * kPer + d % S::kChunkDims / 4, to = queries + set * S::kSetQueries + (m * 32 + warp * 4 + in_seg / S::kPieces) * 16;
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[i] *= unit;
                    uint4 a, b;
                    if (FMT == 1) {
                        split_digits(q, a, b);
                    } else {
                        split<FMT>(q[0], q[1], a.x, a.y);
                        split<FMT>(q[2], q[3], a.z, a.w);
                        split<FMT>(q[4], q[5], b.x, b.y);
                        split<FMT>(q[6], q[7], b.z, b.w);
                    }
                    sts_v4(to, a);
                    sts_v4(to + 512, b);
                }
                if (lane == 0) row_scales[set * kAttentionRows + warp] = row_scale;
            }
            multipliers_sync();
            float row_scale[SETS];
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) row_scale[set] = row_scales[set * kAttentionRows + row];
            uint32_t qa[S::kMmas][4];  // (where registers are short, read again for every tile)
            const auto fetch_query = [&](uint32_t set, uint32_t m) {
                const uint4 w = lds_v4(queries + set * S::kSetQueries + (m * 32 + lane) * 16);
                qa[m][0] = w.x, qa[m][1] = w.y, qa[m][2] = w.z, qa[m][3] = w.w;
            };
            if (S::kQueriesStay)
#pragma unroll
                for (uint32_t m = 0; m < S::kMmas; ++m) fetch_query(0, m);
            Cursor ahead = at;
            more = ahead.next(lengths, p.kv.sequences, g.heads);
            if (kAhead && more) load_query(ahead);
            // tokens of the segment that all rows see, that this row sees, and that exist
            const uint32_t shift = S::kSegs == 1 ? g.tile_shift : 0, end_sub = at.end << shift;
            const int32_t end_token = (int32_t)(end_sub * kTileTokens), existing = min(at.length, end_token);
            const int32_t sure = min(at.length - (int32_t)p.q_tokens + 1, end_token);
            const auto row_of = [&](uint32_t set) { return chunk * S::kRows + set * kAttentionRows + row; };
            int32_t limit[SETS];
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) limit[set] = row_of(set) < g.rows ? min(at.length - (int32_t)p.q_tokens + 1 + (int32_t)(row_of(set) / g.group), end_token) : 0;
            float o[SETS][S::kOwn];  // results: sums of what the tiles' accumulators hold
            float top[SETS], sum[SETS];                          // reference of the row's scores; sum of this lane's weights
            // 8-bit: weights times scales are multiplied by `lift`, a power of two, none yet: 0; and what they may be before that. The lift is kept,
            // not a second reference as a number: it has to follow jumps of the scores, whose difference may leave the range of 32 bits.
            float lift[SETS], most[SETS];
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) {
                top[set] = kNone;
                sum[set] = lift[set] = most[set] = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < S::kOwn; ++i) o[set][i] = 0.f;
            }

            for (uint32_t tile = at.begin << shift; tile < end_sub; tile += S::kSubs) {
                const uint32_t count = min(end_sub - tile, S::kSubs);  // of 16 tokens; this warp's scores are those of warp * kOwnSubs and on
                // ---- scores ----
                mbar_wait(full + turn.slot * 8, turn.phase, limit_ns, p.error_flag);
                float x[SETS][4 * S::kOwnSubs];  // tokens 2 quad, + 1, + 8, + 9 of each 16, row `row`
                float value_scale[SETS][4 * S::kOwnSubs];
#pragma unroll
                for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                    for (uint32_t i = 0; i < 4 * S::kOwnSubs; ++i) x[set][i] = -INFINITY, value_scale[set][i] = 0.f;
                if (warp * S::kOwnSubs < count) {
                    // (the last warp may multiply 16 tokens that are not there; they are left out below)
                    const uint32_t keys = ring + turn.slot * S::kSlot + warp * S::kOwnSubs * S::kSub;
#pragma unroll
                    for (uint32_t n0 = 0; n0 < 2 * S::kOwnSubs; n0 += S::kTogether) {
                        float s[SETS][S::kTogether][4];
                        int upper[SETS][S::kTogether][4], lower[SETS][S::kTogether][4];  // int8: products with digits 3 and 2, and with 1 and 0
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                            for (uint32_t n = 0; n < S::kTogether; ++n)
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[set][n][j] = 0.f, upper[set][n][j] = lower[set][n][j] = 0;
#pragma unroll
                        for (uint32_t seg = 0; seg < S::kSegs; ++seg)
#pragma unroll
                            for (uint32_t c = 0; c < S::kPieces; ++c) {
                                const uint32_t piece = quad * S::kPieces + c, swap = S::kSeg == 128 ? row : row >> 1 & 3u;
                                const uint32_t from = keys + seg * (kTileTokens * S::kSeg) + row * S::kSeg + ((piece ^ swap) << 4);
                                constexpr uint32_t kPer = S::kChunkDims / 4;
                                const uint32_t m = (seg * S::kPieces + c) * kPer;
                                uint32_t word[S::kTogether][S::kWords];
#pragma unroll
                                for (uint32_t n = 0; n < S::kTogether; ++n) {
                                    const uint4 w = lds_v4(from + (n0 + n) / 2 * S::kSub + (n0 + n) % 2 * 8 * S::kSeg);
                                    const uint32_t part[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                    for (uint32_t i = 0; i < 4; ++i) {
                                        if (FMT == 2) e4m3_pairs(part[i], word[n][2 * i % S::kWords], word[n][(2 * i + 1) % S::kWords]);
                                        else word[n][i] = part[i];
                                    }
                                }
#pragma unroll
                                for (uint32_t set = 0; set < SETS; ++set) {
                                    if (!S::kQueriesStay)
#pragma unroll
                                        for (uint32_t i = 0; i < kPer; ++i) fetch_query(set, m + i);
#pragma unroll
                                    for (uint32_t n = 0; n < S::kTogether; ++n)
#pragma unroll
                                        for (uint32_t i = 0; i < kPer; ++i) {
                                            if (FMT == 1) mma_s8s8_16832(i % 2 == 0 ? upper[set][n] : lower[set][n], qa[m + i][0], qa[m + i][1], qa[m + i][2], qa[m + i][3], word[n][i / 2 * 2], word[n][i / 2 * 2 + 1]);
                                            else mma<FMT>(s[set][n], qa[m + i], word[n][2 * i % S::kWords], word[n][(2 * i + 1) % S::kWords]);
                                        }
                                }
                            }
                        const uint32_t sc = scales + turn.slot * S::kScales + warp * S::kOwnSubs * 64 + quad * 8;
#pragma unroll
                        for (uint32_t n = 0; n < S::kTogether; ++n) {
                            uint2 k, v;
                            if (FMT != 0) k = lds_v2(sc + (n0 + n) * 32), v = lds_v2(sc + S::kSubs * 64 + (n0 + n) * 32);
#pragma unroll
                            for (uint32_t set = 0; set < SETS; ++set) {
                                float *const to = x[set] + 2 * (n0 + n), *const scale_to = value_scale[set] + 2 * (n0 + n);
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    if (FMT == 1) to[j] = of_digits(upper[set][n][j], upper[set][n][j + 2], lower[set][n][j], lower[set][n][j + 2]) * row_scale[set];
                                    else to[j] = (s[set][n][j] + s[set][n][j + 2]) * row_scale[set];
                                }
                                if (FMT != 0) {
                                    to[0] *= __uint_as_float(k.x), to[1] *= __uint_as_float(k.y);
                                    scale_to[0] = __uint_as_float(v.x), scale_to[1] = __uint_as_float(v.y);
                                }
                            }
                        }
                    }
                    const int32_t token = (int32_t)((tile + warp * S::kOwnSubs) * kTileTokens);
                    if (attention_some_hidden(token, (int32_t)(S::kOwnSubs * kTileTokens), sure))
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                            for (uint32_t i = 0; i < 4 * S::kOwnSubs; ++i)
                                if (token + (int32_t)(quad * 2 + i % 2 + i / 2 * 8) >= limit[set]) {
                                    x[set][i] = -INFINITY;
                                    value_scale[set][i] = 0.f;  // (it may be anything)
                                }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + turn.slot * 8);
                turn.next();
                // ---- weights ----
                float high[SETS], of_tile[SETS];
#pragma unroll
                for (uint32_t set = 0; set < SETS; ++set) {
                    high[set] = x[set][0];
#pragma unroll
                    for (uint32_t i = 1; i < 4 * S::kOwnSubs; ++i) high[set] = fmaxf(high[set], x[set][i]);
                }
#pragma unroll 1
                for (bool again = false;; again = true) {
                    // as if the references were high enough; if they are not, for any warp, they are raised and all is done again
                    bool raise = false;
#pragma unroll
                    for (uint32_t set = 0; set < SETS; ++set) {
                        float weight[4 * S::kOwnSubs], weight_high = 0.f;
                        of_tile[set] = 0.f;
#pragma unroll
                        for (uint32_t i = 0; i < 4 * S::kOwnSubs; ++i) {
                            weight[i] = exp2_fast(x[set][i] - top[set]);
                            if (FMT != 0) weight_high = fmaxf(weight_high, weight[i] * value_scale[set][i]);
                        }
#pragma unroll
                        for (uint32_t t = 0; t < S::kOwnSubs; ++t) {
                            const uint32_t sub = warp * S::kOwnSubs + t, weights_to = weights_at + set * S::kSetWeights;
                            float w[4];
#pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) {
                                // (weight times scale first: the scale of a token that hardly counts may be far above those that set the lift)
                                w[i] = FMT == 0 ? weight[4 * t + i] : weight[4 * t + i] * value_scale[set][4 * t + i] * lift[set];
                                if (FMT != 0) of_tile[set] += weight[4 * t + i];
                            }
                            uint32_t a[4];
                            if (FMT == 1) {
                                // of two 16s, one MMA's left operand: digits 3 and 2 of the first, of the second; another one's: digits 1 and 0.
                                // What is no number spoils the sum of the weights, and with it the row.
                                weight_digits(w, a);
                                const uint32_t to = weights_to + sub / 2 * 1024 + lane * 16 + sub % 2 * 8;
                                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(a[0]), "r"(a[1]) : "memory");
                                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + 512), "r"(a[2]), "r"(a[3]) : "memory");
#pragma unroll
                                for (uint32_t i = 0; i < 4; ++i)
                                    if (!(w[i] <= Weights<1>::kMost)) of_tile[set] = __uint_as_float(0x7fc00000u);
                            } else {
                                split<FMT>(w[0], w[1], a[0], a[1]);
                                split<FMT>(w[2], w[3], a[2], a[3]);
                                if (FMT == 0) {
                                    // bf16: the weights as they are multiplied, so that they add up to one whatever the halves cut off
#pragma unroll
                                    for (int j = 0; j < 4; j += 2)
                                        of_tile[set] += (__uint_as_float(a[j] << 16) + __uint_as_float(a[j + 1] << 16)) + (__uint_as_float(a[j] & 0xffff0000u) + __uint_as_float(a[j + 1] & 0xffff0000u));
                                }
                                sts_v4(weights_to + (sub * 32 + lane) * 16, make_uint4(a[0], a[1], a[2], a[3]));
                            }
                        }
                        raise = raise || high[set] - top[set] > kHeadroom || (FMT != 0 && weight_high > most[set]);
                    }
                    if (!multipliers_any(!again && raise)) break;
#pragma unroll
                    for (uint32_t set = 0; set < SETS; ++set) {
                        float now = fmaxf(high[set], __shfl_xor_sync(0xffffffffu, high[set], 1));
                        now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 2));
                        if (quad == 0) highs[warp * S::kRows + set * kAttentionRows + row] = now;
                    }
                    multipliers_sync();
                    float keep[SETS], raised[SETS];
#pragma unroll
                    for (uint32_t set = 0; set < SETS; ++set) {
                        float now = -INFINITY;
#pragma unroll
                        for (uint32_t w = 0; w < kWarps; ++w) now = fmaxf(now, highs[w * S::kRows + set * kAttentionRows + row]);
                        keep[set] = 1.f;
                        raised[set] = 0.f;
                        if (now - top[set] > kHeadroom) {
                            now = ceilf(now);
                            raised[set] = now - top[set];
                            keep[set] = exp2_fast(-raised[set]);
                            sum[set] *= keep[set];
                            top[set] = now;
                        }
                    }
                    if (FMT != 0) {
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set) {
                            float weight_high = 0.f;
#pragma unroll
                            for (uint32_t i = 0; i < 4 * S::kOwnSubs; ++i) weight_high = fmaxf(weight_high, exp2_fast(x[set][i] - top[set]) * value_scale[set][i]);
                            weight_high = fmaxf(weight_high, __shfl_xor_sync(0xffffffffu, weight_high, 1));
                            weight_high = fmaxf(weight_high, __shfl_xor_sync(0xffffffffu, weight_high, 2));
                            if (quad == 0) weight_highs[warp * S::kRows + set * kAttentionRows + row] = weight_high;
                        }
                        multipliers_sync();
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set) {
                            float weight_high = 0.f;
#pragma unroll
                            for (uint32_t w = 0; w < kWarps; ++w) weight_high = fmaxf(weight_high, weight_highs[w * S::kRows + set * kAttentionRows + row]);
                            keep[set] = 1.f;
                            if (lift[set] > 0.f || weight_high > 0.f) {
                                // what has been added up stays as it is with a lift of 2^same, unless that is too much for this tile, or for 32 bits
                                const float same = lift[set] > 0.f ? (float)((int)(__float_as_uint(lift[set]) >> 23) - 127) + raised[set] : INFINITY;
                                float next = same;
                                if (same > kMostLift || weight_high * exp2_fast(same) > Weights<FMT>::kMost) {
                                    const int e = (int)(__float_as_uint(weight_high) >> 23) - 126;  // weight_high < 2^e
                                    next = weight_high > 0.f ? fminf((float)(Weights<FMT>::kExponent - e), kMostLift) : kMostLift;
                                    keep[set] = exp2_fast(next - same);
                                }
                                lift[set] = exp2_fast(next);
                            }
                            most[set] = lift[set] > 0.f ? Weights<FMT>::kMost / lift[set] : 0.f;
                        }
                    }
#pragma unroll
                    for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                        for (uint32_t i = 0; i < S::kOwn; ++i) o[set][i] *= keep[set];
                }
#pragma unroll
                for (uint32_t set = 0; set < SETS; ++set) sum[set] += of_tile[set];
                // ---- values: this warp's dimensions, all tokens of the tile ----
                mbar_wait(full + turn.slot * 8, turn.phase, limit_ns, p.error_flag);
                if (warp < S::kValueWarps) {
                    const uint32_t held = ring + turn.slot * S::kSlot;
                    const uint32_t matrix = lane >> 3, line = (lane & 7u) + (matrix & 1u) * 8, swap = S::kSeg == 128 ? line & 7u : line >> 1 & 3u;
                    constexpr uint32_t kPairs = (S::kChunks + 1) / 2;
                    uint32_t from[kPairs];  // in 16 tokens, for each pair of chunks
#pragma unroll
                    for (uint32_t c = 0; c < kPairs; ++c) {
                        const uint32_t piece = warp * S::kChunks + 2 * c + (S::kChunks > 1 ? matrix >> 1 : 0u), seg = piece / (S::kSeg / 16);
                        from[c] = held + seg * (kTileTokens * S::kSeg) + line * S::kSeg + ((piece % (S::kSeg / 16) ^ swap) << 4);
                    }
                    const auto fetch = [&](uint32_t (&v)[kPairs][4], uint32_t t) {
#pragma unroll
                        for (uint32_t c = 0; c < kPairs; ++c) {
                            if (S::kChunks > 1) ldmatrix_x4_trans(v[c], from[c] + t * S::kSub);
                            else ldmatrix_x2_trans(v[c], from[c] + t * S::kSub);
                        }
                    };
                    if constexpr (FMT == 1) {
                        // 32 tokens to an MMA; those without a weight count as nothing whatever their codes are
                        int upper[SETS][S::kAcc][4], lower[SETS][S::kAcc][4];
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                            for (uint32_t i = 0; i < S::kAcc; ++i)
#pragma unroll
                                for (int j = 0; j < 4; ++j) upper[set][i][j] = lower[set][i][j] = 0;
                        const auto add_pair = [&](uint32_t t) {
                            uint4 a[SETS], b[SETS];
#pragma unroll
                            for (uint32_t set = 0; set < SETS; ++set) {
                                const uint32_t weights_of = weights_at + set * S::kSetWeights + (t * 64 + lane) * 16;
                                a[set] = lds_v4(weights_of), b[set] = lds_v4(weights_of + 512);
                            }
                            uint32_t v[kPairs][4], w[kPairs][4];
                            fetch(v, 2 * t);
                            fetch(w, 2 * t + 1);
#pragma unroll
                            for (uint32_t c = 0; c < S::kChunks; ++c) {
                                const uint32_t v0 = v[c / 2][c % 2 * 2], v1 = v[c / 2][c % 2 * 2 + 1], w0 = w[c / 2][c % 2 * 2], w1 = w[c / 2][c % 2 * 2 + 1];
#pragma unroll
                                for (uint32_t i = 0; i < 2; ++i) {
                                    const uint32_t pick = i == 0 ? 0x6420 : 0x7531, b0 = __byte_perm(v0, v1, pick), b1 = __byte_perm(w0, w1, pick);
#pragma unroll
                                    for (uint32_t set = 0; set < SETS; ++set) {
                                        mma_s8s8_16832(upper[set][2 * c + i], a[set].x, a[set].y, a[set].z, a[set].w, b0, b1);
                                        mma_s8s8_16832(lower[set][2 * c + i], b[set].x, b[set].y, b[set].z, b[set].w, b0, b1);
                                    }
                                }
                            }
                        };
                        if (count == S::kSubs) {
#pragma unroll
                            for (uint32_t t = 0; t < S::kSubs / 2; ++t) add_pair(t);
                        } else {
#pragma unroll 1
                            for (uint32_t t = 0; 2 * t < count; ++t) add_pair(t);
                        }
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                            for (uint32_t i = 0; i < S::kOwn; ++i) {
                                const uint32_t m = i / 4 * 2 + i % 2, j = i / 2 % 2;  // dimensions 4 quad ... + 3 of each 16: even, odd, even, odd
                                o[set][i] += of_digits(upper[set][m][j], upper[set][m][j + 2], lower[set][m][j], lower[set][m][j + 2]);
                            }
                    } else {
                        // Accumulators of the upper and lower halves, for one tile: an MMA cuts its sum off, so that it falls short by up to 2^-23 with
                        // every 16 tokens (30,000 tokens in one accumulator were off by 1.6e-4, with a sum a tile it is 2^-24 for its addition).
                        float acc[SETS][S::kAcc][4];
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                            for (uint32_t i = 0; i < S::kAcc; ++i) acc[set][i][0] = acc[set][i][1] = acc[set][i][2] = acc[set][i][3] = 0.f;
                        const auto add_sub = [&](uint32_t t, bool edge) {
                            uint32_t wa[SETS][4];
#pragma unroll
                            for (uint32_t set = 0; set < SETS; ++set) {
                                const uint4 w = lds_v4(weights_at + set * S::kSetWeights + (t * 32 + lane) * 16);
                                wa[set][0] = w.x, wa[set][1] = w.y, wa[set][2] = w.z, wa[set][3] = w.w;
                            }
                            uint32_t v[kPairs][4];
                            fetch(v, t);
                            const int32_t first = (int32_t)((tile + t) * kTileTokens);
                            if (edge) {
                                // Rows behind the sequence's end hold anything: zeros are taken for them. Among draft tokens a value that is not
                                // finite may be seen by some rows only, and a weight of zero does not take it out of a sum: it is taken out
                                // here and added to the rows that see it.
                                bool odd = false;
#pragma unroll
                                for (uint32_t c = 0; c < kPairs; ++c)
#pragma unroll
                                    for (uint32_t i = 0; i < (S::kChunks > 1 ? 4 : 2); ++i) {
                                        const int32_t k = first + (int32_t)(quad * 2 + i % 2 * 8);
                                        v[c][i] &= (k < existing ? 0xffffu : 0u) | (k + 1 < existing ? 0xffff0000u : 0u);
                                        if (p.q_tokens > 1)
#pragma unroll
                                            for (int b = 0; b < 4; b += FMT == 0 ? 2 : 1)
                                                if (not_finite<FMT>(v[c][i], b)) {
                                                    odd = true;
                                                    v[c][i] &= ~((FMT == 0 ? 0xffffu : 0xffu) << (b * 8));
                                                }
                                    }
                                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                                    for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll 1
                                        for (int32_t k = 0; k < (int32_t)kTileTokens && first + k < limit[set]; ++k) {
                                            const uint32_t turned = S::kSeg == 128 ? (uint32_t)k & 7u : (uint32_t)k >> 1 & 3u, at_token = held + t * S::kSub + (uint32_t)k * S::kSeg;
#pragma unroll
                                            for (uint32_t i = 0; i < S::kAcc; ++i)
#pragma unroll
                                                for (uint32_t j = 0; j < 2; ++j) {
                                                    const uint32_t d = warp * S::kWarpDims + (FMT == 0 ? i * 8 + quad * 2 + j : i / 2 * 16 + quad * 4 + j * 2 + (i & 1u));
                                                    const uint32_t byte = d * (FMT == 0 ? 2 : 1), piece = byte % S::kSeg / 16;
                                                    const uint32_t e = lds_u32((at_token + byte / S::kSeg * (kTileTokens * S::kSeg) + ((piece ^ turned) << 4) + byte % 16) & ~3u);
                                                    if (not_finite<FMT>(e, byte & 3u)) acc[set][i][j] += FMT == 0 ? __uint_as_float((e >> ((byte & 3u) * 8)) << 16) : __uint_as_float(0x7fc00000u);
                                                }
                                        }
                                    __syncwarp();
                                }
                            }
#pragma unroll
                            for (uint32_t c = 0; c < S::kChunks; ++c) {
                                const uint32_t b0 = v[c / 2][c % 2 * 2], b1 = v[c / 2][c % 2 * 2 + 1];
                                if (FMT == 0) {
#pragma unroll
                                    for (uint32_t set = 0; set < SETS; ++set) mma<FMT>(acc[set][c], wa[set], b0, b1);
                                } else {
                                    uint32_t even[2], odd[2];
                                    e4m3_pairs(__byte_perm(b0, 0, 0x3120), even[0], odd[0]);
                                    e4m3_pairs(__byte_perm(b1, 0, 0x3120), even[1], odd[1]);
#pragma unroll
                                    for (uint32_t set = 0; set < SETS; ++set) {
                                        mma<FMT>(acc[set][2 * c], wa[set], even[0], even[1]);
                                        mma<FMT>(acc[set][2 * c + 1], wa[set], odd[0], odd[1]);
                                    }
                                }
                            }
                        };
                        const uint32_t plain = (uint32_t)max(min(sure - (int32_t)(tile * kTileTokens), (int32_t)(count * kTileTokens)), 0) / kTileTokens;  // 16s that all rows see
                        if (plain == S::kSubs) {
#pragma unroll
                            for (uint32_t t = 0; t < S::kSubs; ++t) add_sub(t, false);
                        } else {
#pragma unroll 1
                            for (uint32_t t = 0; t < count; ++t) add_sub(t, t >= plain);
                        }
#pragma unroll
                        for (uint32_t set = 0; set < SETS; ++set)
#pragma unroll
                            for (uint32_t i = 0; i < S::kOwn; ++i) {
                                const uint32_t m = FMT == 0 ? i / 2 : i / 4 * 2 + i % 2, j = FMT == 0 ? i % 2 : i / 2 % 2;
                                o[set][i] += acc[set][m][j] + acc[set][m][j + 2];
                            }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + turn.slot * 8);
                turn.next();
                weights_at = weights_at == weights ? weights + S::kWeights : weights;
            }

            // ---- the segment's result ----
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) {
                sum[set] += __shfl_xor_sync(0xffffffffu, sum[set], 1);
                sum[set] += __shfl_xor_sync(0xffffffffu, sum[set], 2);
                if (quad == 0) sums[warp * S::kRows + set * kAttentionRows + row] = sum[set];
            }
            multipliers_sync();
            const bool whole = at.whole_item();
            uint32_t owner = 0, contributors = 0;
            if (!whole) at.contributors(share.cut, blockIdx.x, &owner, &contributors);
            float *const part = p.parts + ((uint64_t)blockIdx.x * 2 + (blockIdx.x == owner ? 1 : 0)) * kPart;
            constexpr uint32_t kBeside = FMT == 0 ? 2 : 4;  // numbers beside each other
            const auto dim_of = [&](uint32_t i) { return warp * S::kWarpDims + i / kBeside * (4 * kBeside) + quad * kBeside + i % kBeside; };
#pragma unroll
            for (uint32_t set = 0; set < SETS; ++set) {
                // numbers of the row: bf16: dimensions 8 i + 2 quad, + 1; 8-bit: 16 i + 4 quad ... + 3, from the warp's first on
                const uint32_t in_item = set * kAttentionRows + row, r = row_of(set);
                const bool holds = r < g.rows && warp < S::kValueWarps;
                float mine[S::kOwn];
                {
                    const float unlift = FMT == 0 ? 1.f : lift[set] > 0.f ? 1.f / lift[set] : 0.f;
#pragma unroll
                    for (uint32_t i = 0; i < S::kOwn; ++i) mine[i] = o[set][i] * unlift;
                }
                float total = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) total += sums[w * S::kRows + in_item];
                if (!whole) {
                    // ---- a partial result; the block that is the last to leave one of an item joins them below ----
                    if (holds)
#pragma unroll
                        for (uint32_t i = 0; i < S::kOwn; i += kBeside) {
                            float *const to = part + in_item * HDP + dim_of(i);
                            if (FMT == 0) *reinterpret_cast<float2 *>(to) = make_float2(mine[i], mine[i + 1]);
                            else *reinterpret_cast<float4 *>(to) = make_float4(mine[i], mine[i + 1], mine[(i + 2) % S::kOwn], mine[(i + 3) % S::kOwn]);
                        }
                    if (warp == 0 && quad == 0) {
                        part[S::kRows * HDP + in_item] = top[set] == kNone ? -INFINITY : top[set];
                        part[S::kRows * (HDP + 1) + in_item] = total;
                    }
                } else if (holds) {
                    const bool none = at.length - (int32_t)p.q_tokens + 1 + (int32_t)(r / g.group) <= 0;
                    const float by = 1.f / total;
                    const uint64_t base = ((uint64_t)at.s * p.q_tokens + r / g.group) * p.out_stride + ((uint64_t)head * g.group + r % g.group) * p.kv.head_dim;
#pragma unroll
                    for (uint32_t i = 0; i < S::kOwn; ++i) mine[i] = none ? 0.f : mine[i] * by;
#pragma unroll
                    for (uint32_t i = 0; i < S::kOwn; i += kBeside) {
                        const uint32_t d = dim_of(i);
                        if (d >= p.kv.head_dim) continue;
                        if (p.out_is_f32) {
                            float *const to = static_cast<float *>(p.out) + base + d;
                            if (FMT == 0) *reinterpret_cast<float2 *>(to) = make_float2(mine[i], mine[i + 1]);
                            else *reinterpret_cast<float4 *>(to) = make_float4(mine[i], mine[i + 1], mine[(i + 2) % S::kOwn], mine[(i + 3) % S::kOwn]);
                        } else {
                            uint16_t *const to = static_cast<uint16_t *>(p.out) + base + d;
                            if (FMT == 0) *reinterpret_cast<uint32_t *>(to) = pack_bf16(mine[i], mine[i + 1]);
                            else *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16(mine[i], mine[i + 1]), pack_bf16(mine[(i + 2) % S::kOwn], mine[(i + 3) % S::kOwn]));
                        }
                    }
                }
            }
            if (!whole) {
                __threadfence();
                multipliers_sync();
                if (threadIdx.x == 0) {
                    uint32_t *const to = joins + left_parts * 6;
                    const bool last = atomicAdd(p.counters + owner, 1u) + 1 == contributors;
                    if (last) {
                        __threadfence();  // the others' partial results are read behind the barrier below
                        p.counters[owner] = 0;
                    }
                    to[0] = last, to[1] = owner, to[2] = contributors, to[3] = at.s, to[4] = at.item, to[5] = (uint32_t)at.length;
                }
                ++left_parts;
            }
            at = ahead;
        } while (more);

        // ---- partial results of cut items that are complete, joined in the order of the tiles ----
        // They come by bulk copies into the ring, which is free now: plain loads took 14000 cycles for 36 pieces of 6 KB, copies 3000. (Adding up a first
        // half or quarter while the others arrive was slower: 13.7 us in place of 13.1 for 8200 tokens.)
        multipliers_sync();
        uint32_t phase = 0;
#pragma unroll 1
        for (uint32_t n = 0; n < left_parts; ++n) {
            const uint32_t *const job = joins + n * 6;
            if (!job[0]) continue;
            const uint32_t owner = job[1], contributors = job[2], seq = job[3], head = job[4] / g.chunks, chunk = job[4] % g.chunks;
            const uint32_t rows = min(g.rows - chunk * S::kRows, S::kRows), bytes = rows * HDP * 4;
            // the pieces lie from the ring's start on, factors [piece][row] behind them, in what was there for scales, weights and queries
            const uint32_t factors_at = full - contributors * S::kRows * 4, room = (factors_at - ring) / bytes;
            float *const factors = reinterpret_cast<float *>(shared_raw + (factors_at - raw));
            // piece k lies 2 k - 1 places behind the owner's, which is the first one
            const float *const first = p.parts + ((uint64_t)owner * 2 + 1) * kPart;
            const auto piece = [&](uint32_t k) { return first + (k == 0 ? 0 : 2 * k - 1) * kPart; };
            float4 sums_of[2 * SETS];  // 16 bytes of the item's rows, and those 256 x 16 behind them
#pragma unroll
            for (uint32_t j = 0; j < 2 * SETS; ++j) sums_of[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (uint32_t done = 0; done < contributors; done += room) {
                const uint32_t now = min(room, contributors - done);
                if (done) multipliers_sync();  // those before have been read
                if (threadIdx.x == 0) mbar_expect(joined, now * bytes);
                for (uint32_t k = threadIdx.x; k < now; k += kMultipliers) {
                    asm volatile("fence.proxy.async;" ::: "memory");
                    copy_bytes(ring + k * bytes, piece(done + k), bytes, joined);
                }
                if (done == 0) {
                    // a warp for each row; pieces that saw nothing have zeros, rows whose scores are NaNs keep those
#pragma unroll 1
                    for (uint32_t of = warp; of < S::kRows; of += kWarps) {
                        float best = -INFINITY, total = 0.f, t[kMostBlocks / 32], l[kMostBlocks / 32];
#pragma unroll
                        for (uint32_t i = 0; i < kMostBlocks / 32; ++i) {
                            const uint32_t k = lane + i * 32;
                            t[i] = k < contributors ? __ldcg(piece(k) + S::kRows * HDP + of) : -INFINITY;
                            l[i] = k < contributors ? __ldcg(piece(k) + S::kRows * (HDP + 1) + of) : 0.f;
                        }
#pragma unroll
                        for (uint32_t i = 0; i < kMostBlocks / 32; ++i) best = fmaxf(best, t[i]);
#pragma unroll
                        for (int off = 16; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, off));
#pragma unroll
                        for (uint32_t i = 0; i < kMostBlocks / 32; ++i) {
                            const float f = t[i] == -INFINITY ? 0.f : exp2_fast(t[i] - best);
                            total += t[i] == -INFINITY ? l[i] : l[i] * f;
                            if (lane + i * 32 < contributors) factors[(lane + i * 32) * S::kRows + of] = f;
                        }
#pragma unroll
                        for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
                        if (lane == 0) sums[of] = total;
                    }
                    multipliers_sync();
                }
                mbar_wait(joined, phase, limit_ns, p.error_flag);
                phase ^= 1u;
#pragma unroll
                for (uint32_t j = 0; j < 2 * SETS; ++j) {
                    const uint32_t i = threadIdx.x + j * kMultipliers;
                    if (i * 16 >= bytes) continue;
                    const uint32_t of = i / (HDP / 4);
                    float4 o4 = sums_of[j];
#pragma unroll 4
                    for (uint32_t k = 0; k < now; ++k) {
                        const uint4 w = lds_v4(ring + k * bytes + i * 16);
                        const float f = factors[(done + k) * S::kRows + of];
                        o4.x = fmaf(__uint_as_float(w.x), f, o4.x), o4.y = fmaf(__uint_as_float(w.y), f, o4.y);
                        o4.z = fmaf(__uint_as_float(w.z), f, o4.z), o4.w = fmaf(__uint_as_float(w.w), f, o4.w);
                    }
                    sums_of[j] = o4;
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < 2 * SETS; ++j) {
                const uint32_t i = threadIdx.x + j * kMultipliers, of = i / (HDP / 4), d = i % (HDP / 4) * 4;
                if (i * 16 >= bytes || d >= p.kv.head_dim) continue;
                const uint32_t r = chunk * S::kRows + of;
                const bool none = (int32_t)job[5] - (int32_t)p.q_tokens + 1 + (int32_t)(r / g.group) <= 0;
                const float by = 1.f / sums[of];
                const float4 v = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sums_of[j].x * by, sums_of[j].y * by, sums_of[j].z * by, sums_of[j].w * by);
                const uint64_t to = ((uint64_t)seq * p.q_tokens + r / g.group) * p.out_stride + ((uint64_t)head * g.group + r % g.group) * p.kv.head_dim + d;
                if (p.out_is_f32) *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + to) = v;
                else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
            }
            multipliers_sync();  // factors and sums have been read
        }
    }

    // ---- sequences without tokens ----
    for (uint32_t s = blockIdx.x; s < p.kv.sequences; s += gridDim.x) {
        if (__ldcg(p.lengths + s) > 0) continue;
        const uint32_t width = p.heads * p.kv.head_dim / 4;
        for (uint32_t i = threadIdx.x; i < width * p.q_tokens; i += kThreads) {
            const uint64_t to = ((uint64_t)s * p.q_tokens + i / width) * p.out_stride + (uint64_t)(i % width) * 4;
            if (p.out_is_f32) *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + to) = make_float4(0.f, 0.f, 0.f, 0.f);
            else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + to) = make_uint2(0u, 0u);
        }
    }
}

// ---- host ----

// Rows of the cache as [page][head][token][value], or [page][head][segment][token][value in it]; copies of a tile's tokens by
// one segment, or all.
template <int FMT, int HDP>
bool encode_map(EncodeTiledFn encode, CUtensorMap *map, const KvView &kv, const uint8_t *pool, bool whole_rows, uint32_t tile_shift) {
    using S = Shape<FMT, HDP, 1>;
    constexpr uint32_t kSegValues = S::kSeg / (FMT == 0 ? 2 : 1);
    const CUtensorMapDataType type = FMT == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUtensorMapSwizzle swizzle = S::kSeg == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    if (whole_rows && S::kSegs > 1) {
        const cuuint64_t dims[5] = {kSegValues, kv.page_tokens, kv.head_dim / kSegValues, kv.kv_heads, kv.pages};
        const cuuint64_t strides[4] = {kv.token_stride, S::kSeg, kv.head_stride, kv.page_stride};
        const cuuint32_t box[5] = {kSegValues, kTileTokens, S::kSegs, 1, 1};
        return encode(map, type, 5, const_cast<uint8_t *>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    const cuuint64_t dims[4] = {kv.head_dim, kv.page_tokens, kv.kv_heads, kv.pages};
    const cuuint64_t strides[3] = {kv.token_stride, kv.head_stride, kv.page_stride};
    const cuuint32_t box[4] = {kSegValues, kTileTokens << tile_shift, 1, 1};
    return encode(map, type, 4, const_cast<uint8_t *>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, int HDP, int SETS>
cudaError_t launch(const AttentionParams &p, uint32_t sm_count, cudaStream_t stream) {
    using S = Shape<FMT, HDP, SETS>;
    const EncodeTiledFn encode = encode_tiled_fn();
    CUtensorMap maps[2];
    // Rows of one segment come 64 tokens at a time where pages allow (smaller copies are more than the copy engine takes; larger ones would
    // bring more of what lies behind a sequence's end).
    uint32_t shift = 0;
    while (S::kSegs == 1 && shift < 2 && p.kv.page_tokens % (2 * kTileTokens << shift) == 0) ++shift;
    const bool whole_rows = p.kv.head_dim * (FMT == 0 ? 2 : 1) % S::kSeg == 0;
    if (!encode || !encode_map<FMT, HDP>(encode, &maps[0], p.kv, p.kv.k, whole_rows, shift) || !encode_map<FMT, HDP>(encode, &maps[1], p.kv, p.kv.v, whole_rows, shift)) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> ready{0};  // a bit for each device: the attribute is the kernel's, once set it stays
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(attention_kernel<FMT, HDP, SETS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kShared);
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    Geometry g;
    g.group = p.heads / p.kv.kv_heads;
    g.rows = g.group * p.q_tokens;
    g.chunks = (g.rows + S::kRows - 1) / S::kRows;
    g.heads = p.kv.kv_heads * g.chunks;
    g.tile_shift = shift;
    g.pages = attention_pages(p.kv.page_tokens, shift);
    g.whole_rows = whole_rows || S::kSegs == 1;
    return launch_dependent(attention_kernel<FMT, HDP, SETS>, dim3(sm_count < kMostBlocks ? sm_count : kMostBlocks), kThreads, S::kShared, stream, p, g, maps[0], maps[1]);
}

// Eights of rows that an item has together read and convert every key and value once; each has more registers and less of the ring. Measured on
// 51,000 tokens in four sequences, 4 key heads, us with 1 / 2 / 3 eights an item: bf16 of 256 with 12 rows 49 / 44 / 51, with 24 rows
// 75 / 64 / 55; bf16 of 128 with 32 rows 46 / 42 / 52; e4m3 of 128 with 16 rows 34 / 26 / 35, with 32 rows 52 / 40 / 57; int8 of 128 with 16 rows
// 32 / 28 / 38; of 64 with 16 rows bf16 27 / 21 / 26, e4m3 31 / 22 / 26, int8 31 / 23 / 30; of 256 with 24 rows int8 63 / 67 / 60, e4m3 62 / 58 / 62:
// there the digits, or fp16 pairs, of more rows do not fit the registers, and one eight is kept. More rows of bf16 of 256, 2 / 3 eights an item:
// 40 and 48 rows 104 / 87, 56 and 72 rows 125 to 133 / 143, 80 rows 128 to 142 / 146, 88 rows 175 / 146: how the items fall on the blocks counts as
// much as their width, and the rule is on the wrong side by up to a fifth at 48, 56 and 72 rows. (Bf16 of 256 with three
// eights spills 104 bytes.)
template <int FMT, int HDP>
cudaError_t launch_sets(const AttentionParams &p, uint32_t sm_count, cudaStream_t stream) {
    const uint32_t sets = (p.heads / p.kv.kv_heads * p.q_tokens + kAttentionRows - 1) / kAttentionRows;
    if constexpr (FMT == 0 || HDP < 256) {
        if constexpr (HDP == 256)
            if (sets > 1 && sets % 2 == 1) return launch<FMT, HDP, 3>(p, sm_count, stream);
        if (sets > 1) return launch<FMT, HDP, 2>(p, sm_count, stream);
    }
    return launch<FMT, HDP, 1>(p, sm_count, stream);
}

template <int FMT>
cudaError_t launch_dim(const AttentionParams &p, uint32_t sm_count, cudaStream_t stream) {
    if (p.kv.head_dim <= 64) return launch_sets<FMT, 64>(p, sm_count, stream);
    if (p.kv.head_dim <= 128) return launch_sets<FMT, 128>(p, sm_count, stream);
    return launch_sets<FMT, 256>(p, sm_count, stream);
}

}  // namespace q4

extern "C" size_t q4k_attention_part_floats(uint32_t sm_count) { return (size_t)sm_count * 2 * q4::kMostSets * q4::kAttentionRows * (q4::kMaxHeadDim + 2); }

extern "C" cudaError_t q4k_attention(const q4::AttentionParams *p, uint32_t sm_count, cudaStream_t stream) {
    if (p->kv.format == 0u) return q4::launch_dim<0>(*p, sm_count, stream);
    if (p->kv.format == 1u) return q4::launch_dim<1>(*p, sm_count, stream);
    return q4::launch_dim<2>(*p, sm_count, stream);
}
