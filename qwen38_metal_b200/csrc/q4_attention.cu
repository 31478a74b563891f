// Attention of new tokens over a paged cache. Counterparts in the reference: the cache's scores and values kernels
// (src/metal_runtime.rs:8230-8798, shaders/qwen38.metal:4761-5323).
//
//     out = sum_j p_j v_j / sum_j p_j,   p_j = e^(scale q.k_j)
//
// Every key and value is read once from memory for eight query rows (token, head) that share its key head: at one byte a value that is
// 12 to 16 operations a byte, so memory is the bound, and the kernel is built around keeping loads in flight.
//
//   * One block per SM, eight warps, each with a ring of its own in shared memory. Tiles of 16 tokens (they never cross a page)
//     go round the warps, two at a time for 8-bit caches; a warp asks for keys and values of its next tiles with tensor copies, past the
//     end of an item too, so that 190 KB stay in flight per SM while results are joined. No warp waits for another one inside an item.
//   * Both products run on m16n8k16 MMAs with eight query rows: rows 0...7 of the left operand hold the upper halves of the eight
//     rows' factors, rows 8...15 the lower halves, so that the sum of the two accumulators is a product of factors of 16 bits or more
//     (two bf16 numbers, error 2^-17; two fp16 numbers for 8-bit caches, 2^-22), at no cost: the rows would be empty.
//   * Queries against int8 keys run on whole-number MMAs as they lie in memory, four 8-bit digits of every query; other 8-bit codes become
//     fp16 exactly. Which dimensions an MMA multiplies is free as long as queries and keys agree, so that a lane takes whole 16-byte pieces
//     of a key row; values are read transposed as pairs of bytes, which gives the lane a pair of dimensions, one for each of two MMAs.
//   * One pass: every warp keeps a sum and a result of each row in registers, relative to a power of two that is raised when a score lies 8
//     above it, which is seldom after the first tiles (raising it with every maximum cost 128 multiplications a tile). The scale of a
//     token's values goes into its weight; weights times scales have a reference of their own, so that they stay in fp16's range
//     whatever the scales are.
//   * The work of all sequences is cut into equal shares by every block for itself (q4_attention_plan.h), from the lengths in device memory:
//     a captured graph follows them. Results of an item cut over several blocks are joined in order by the last one.
#include <cuda_fp8.h>

#include <atomic>

#include "q4_attention.h"
#include "q4_attention_plan.h"
#include "q4_device.cuh"
#include "q4_tensor_map.h"

namespace q4 {

constexpr uint32_t kWarps = 8, kThreads = kWarps * 32;
constexpr uint32_t kRoundDims = 64;             // dimensions joined at a time
constexpr uint32_t kRoundPitch = kRoundDims + 16;  // floats between rows of the join buffer: lanes of a store fall into different banks
constexpr uint32_t kLeastRun = 16;              // tiles: shorter runs cost more in joining than they save
constexpr float kNone = -3.0e38f;               // a reference below all scores: the row has seen nothing
constexpr float kHeadroom = 8.f;                // how far above its reference a score may lie, in powers of two
// 8-bit caches: a weight times scale is brought to 2^11 when it becomes the reference and may grow to 2^15, near the end of fp16's
// range, so that lower halves keep 16 bits of weights down to 2^-19 of the largest one (and 2^-35 of it below)
constexpr int kWeightExponent = 11;
constexpr float kMostWeight = 32768.f;
constexpr unsigned long long kWaitLimitNs = 200ull * 1000 * 1000, kLateLimitNs = 1000 * 1000;
constexpr uint32_t kSharedLimit = 227 * 1024;

template <int FMT, int HDP>
struct Shape {
    static constexpr uint32_t kRow = HDP * (FMT == 0 ? 2 : 1);       // bytes of a token's row in shared memory
    static constexpr uint32_t kSeg = kRow < 128 ? kRow : 128;        // bytes of it that one copy brings
    static constexpr uint32_t kSegs = kRow / kSeg;
    static constexpr uint32_t kTile = kTileTokens * kRow;            // a tile of keys or of values
    static constexpr uint32_t kPieces = kSeg / 64;                   // 16-byte pieces of a segment a lane takes from a key row
    static constexpr uint32_t kMmas = HDP / 16;                      // per 8 tokens of scores
    static constexpr uint32_t kChunks = kRow / 16;                   // 16-byte pieces of a row
    static constexpr uint32_t kChunkDims = FMT == 0 ? 8 : 16;
    static constexpr uint32_t kAcc = HDP / 8;                        // accumulators of four numbers
    static constexpr uint32_t kStep = FMT == 0 ? 1 : 2;              // tiles a warp multiplies at a time
    // shared memory: rings, their scales, barriers, queries, the join buffer, and small arrays
    static constexpr uint32_t kQueries = kMmas * 32 * 16;
    static constexpr uint32_t kJoin = kWarps * kAttentionRows * kRoundPitch * 4;
    static constexpr uint32_t kSmall = 2048;
    static constexpr uint32_t kSlot = kStep * kTile, kSlotScales = kStep * 64;
    static constexpr uint32_t kFit = (kSharedLimit - 1024 - kQueries - kJoin - kSmall) / (kWarps * (kSlot + kSlotScales + 8));
    static constexpr uint32_t kSlots = kFit < 8 ? kFit : 8;          // of a warp's ring: keys and values of its steps in turn
    static constexpr uint32_t kRing = kWarps * kSlots * kSlot, kScales = kWarps * kSlots * kSlotScales, kBars = (kWarps * kSlots * 8 + 15) / 16 * 16;
    static constexpr uint32_t kShared = 1024 + kRing + kScales + kBars + kQueries + kJoin + kSmall;
    static_assert(kSlots >= 2 && kStep * (kSegs + 1) <= 32, "");
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

// Bytes 0 and 2, and bytes 1 and 3, of a word of int8 codes as fp16: 0x6400 | u is 1024 + u, with u = code + 128.
__device__ __forceinline__ uint32_t int8_even(uint32_t w) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"((w & 0x00ff00ffu) ^ 0x64806480u), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {  // the lower two bytes
    uint32_t r;
    asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
    return r;
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
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

__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int token, int head, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(token),
                 "r"(head), "r"(page)
                 : "memory");
}
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// ---- a block's share ----

struct Geometry {
    uint32_t chunks;  // items of a key head: eight query rows each
    uint32_t heads;   // items of a sequence = key heads * chunks
    uint32_t rows;    // query rows of a key head
    uint32_t group;   // query heads of a key head
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

__device__ __forceinline__ uint64_t warp_scan(uint64_t v, uint32_t lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint64_t o = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= (uint32_t)off) v += o;
    }
    return v;
}

// All threads. `scratch`: 3 * kWarps + 2 words of 64 bits in shared memory. Up to 32 sequences every warp finds it by itself.
__device__ __forceinline__ Share share_of_block(const AttentionParams &p, const Geometry &g, uint64_t *scratch) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, sequences = p.kv.sequences;
    const bool few = sequences <= 32;
    const uint32_t mine = few ? lane : threadIdx.x, stride = few ? 32 : kThreads;
    uint64_t tiles = 0;
    uint32_t items = 0, longest = 0, own = 0;  // own: tiles of the thread's first sequence
    for (uint32_t s = mine; s < sequences; s += stride) {
        const int64_t raw = __ldcg(p.lengths + s), most = (int64_t)p.kv.per_sequence * p.kv.page_tokens, n = raw < 0 ? 0 : raw > most ? most : raw;
        if (raw != n && blockIdx.x == 0) *p.kv.input_error = 1;
        const uint32_t t = attention_tiles(n);
        if (s == mine) own = t;
        tiles += t;
        items += t > 0;
        longest = max(longest, t);
    }
    uint64_t scan = warp_scan(tiles, lane);
    tiles = __shfl_sync(0xffffffffu, scan, 31);
    items = __reduce_add_sync(0xffffffffu, items);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (!few) {
        if (lane == 0) scratch[warp] = tiles, scratch[kWarps + warp] = items, scratch[2 * kWarps + warp] = longest;
        __syncthreads();
        tiles = items = longest = 0;
        for (uint32_t w = 0; w < kWarps; ++w) {
            tiles += scratch[w];
            items += (uint32_t)scratch[kWarps + w];
            longest = max(longest, (uint32_t)scratch[2 * kWarps + w]);
        }
    }
    Share share;
    share.any = false;
    share.at = Cursor{};
    if (tiles == 0) return share;
    share.cut = attention_cut(tiles * g.heads, (uint64_t)items * g.heads, longest, gridDim.x, kLeastRun);
    const AttentionCut &cut = share.cut;
    const uint64_t target = attention_target(cut, blockIdx.x);
    if (cut.mode != kEqualPieces && target >= cut.tiles) return share;
    // the sequence that holds piece or tile number `target`
    uint64_t start = 0;
    uint32_t s = 0;
    bool found = false;
    if (few) {
        const uint64_t weight = attention_weight(cut, own, g.heads), to = warp_scan(weight, lane);
        const uint32_t hit = __ballot_sync(0xffffffffu, target >= to - weight && target < to);
        found = hit != 0;
        s = found ? __ffs(hit) - 1 : 0;
        start = __shfl_sync(0xffffffffu, to - weight, s);
    } else {
        uint64_t before = 0;
        for (uint32_t base = 0; base < sequences && !found; base += kThreads) {
            const uint32_t i = base + threadIdx.x;
            const uint32_t t = base == 0 ? own : i < sequences ? attention_tiles(length_of(p, i)) : 0u;
            const uint64_t weight = attention_weight(cut, t, g.heads);
            const uint64_t to = warp_scan(weight, lane);
            __syncthreads();
            if (lane == 31) scratch[warp] = to;
            if (threadIdx.x == 0) scratch[kWarps] = ~0ull;
            __syncthreads();
            uint64_t from = before + to - weight;
            for (uint32_t w = 0; w < kWarps; ++w) {
                if (w < warp) from += scratch[w];
                before += scratch[w];
            }
            if (target >= from && target < from + weight) scratch[kWarps] = i, scratch[kWarps + 1] = from;
            __syncthreads();
            found = scratch[kWarps] != ~0ull;
            s = (uint32_t)scratch[kWarps];
            start = scratch[kWarps + 1];
        }
        __syncthreads();
    }
    if (found) share.any = share.at.start(cut, target, s, start, [&](uint32_t i) { return length_of(p, i); }, sequences, g.heads);
    return share;
}

// ---- asking for tiles ----

// What a warp asks for, ahead of what it multiplies: keys of its next kStep tiles into one slot, then their values into the next.
// Lane i * kSegs + j brings segment j of tile i, the lanes behind those the scales. Page numbers are read one step ahead. A step's
// second tile may lie behind the segment's end: such a copy starts outside the tensor map and brings zeros.
template <int FMT, int HDP>
struct Asker {
    using S = Shape<FMT, HDP>;
    static constexpr uint32_t kCopies = S::kStep * S::kSegs;
    Cursor at;
    uint32_t tile, head, slot, page, place;  // page and place: of this lane's tile
    bool more, values;

    __device__ __forceinline__ static uint32_t mine(uint32_t lane) { return lane < kCopies ? lane / S::kSegs : (lane - kCopies) % S::kStep; }
    __device__ __forceinline__ void look(const AttentionParams &p, const Geometry &g, uint32_t warp, uint32_t lane) {
        while (tile >= at.end) {
            if (!at.next([&](uint32_t i) { return length_of(p, i); }, p.kv.sequences, g.heads)) {
                more = false;
                return;
            }
            tile = at.begin + warp * S::kStep;
            head = g.chunks == 1 ? at.item : at.item / g.chunks;
        }
        const uint32_t t = tile + mine(lane), entry = g.pages.page_of(t);
        place = (t - entry * g.pages.per) * kTileTokens;
        page = t < at.end ? (uint32_t)__ldcg(p.kv.table + (uint64_t)at.s * p.kv.row_stride + entry) : ~0u;
    }
    __device__ __forceinline__ void start(const Share &share, const AttentionParams &p, const Geometry &g, uint32_t warp, uint32_t lane) {
        at = share.at;
        tile = at.begin + warp * S::kStep;
        head = at.item / g.chunks;
        slot = 0;
        more = true;
        values = false;
        look(p, g, warp, lane);
    }
    __device__ __forceinline__ void ask(const AttentionParams &p, const Geometry &g, const CUtensorMap *k_map, const CUtensorMap *v_map, uint32_t ring, uint32_t scales, uint32_t bars,
                                        uint32_t warp, uint32_t lane) {
        if (!more) return;
        const uint32_t bar = bars + slot * 8;
        const bool there = page < p.kv.pages;
        const uint32_t absent = __ballot_sync(0xffffffffu, !there);
        uint32_t bytes = S::kSlot + (FMT == 0 ? 0u : S::kSlotScales);
        if (absent) {
            // behind the segment's end, or no page of the cache
            if (!there && tile + mine(lane) < at.end) *p.kv.input_error = 1;
            if (FMT != 0) {
                bytes -= 64 * __popc(absent >> kCopies & ((1u << S::kStep) - 1));
                if (!there && lane >= kCopies && lane < kCopies + S::kStep) {
                    for (uint32_t i = 0; i < 64; i += 16) sts_v4(scales + slot * S::kSlotScales + (lane - kCopies) * 64 + i, make_uint4(0u, 0u, 0u, 0u));
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
            }
        }
        if (lane == 0) mbar_expect(bar, bytes);
        if (lane < kCopies)
            copy_tile(ring + slot * S::kSlot + lane * (kTileTokens * S::kSeg), values ? v_map : k_map, bar, (int)(lane % S::kSegs * S::kSeg / (FMT == 0 ? 2 : 1)), (int)place, (int)head,
                      (int)(there ? page : p.kv.pages));
        else if (FMT != 0 && lane < kCopies + S::kStep && there)
            copy_bytes(scales + slot * S::kSlotScales + (lane - kCopies) * 64, (values ? p.kv.v_scales : p.kv.k_scales) + ((uint64_t)page * p.kv.kv_heads + head) * p.kv.page_tokens + place, 64, bar);
        slot = slot + 1 == S::kSlots ? 0 : slot + 1;
        if (values) {
            tile += kWarps * S::kStep;
            look(p, g, warp, lane);
        }
        values = !values;
    }
};

template <int FMT>
__device__ __forceinline__ bool not_finite(uint32_t w, uint32_t byte) {  // the value that begins at this byte of a word
    if (FMT == 0) return ((w >> (byte * 8)) & 0x7f80u) == 0x7f80u;
    return ((w >> (byte * 8)) & 0x7fu) == 0x7fu;
}

// ---- the kernel ----

template <int FMT, int HDP>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ Geometry g, const __grid_constant__ CUtensorMap k_map,
                                                                const __grid_constant__ CUtensorMap v_map) {
    using S = Shape<FMT, HDP>;
    constexpr uint32_t kStep = S::kStep;
    extern __shared__ uint8_t shared_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(shared_raw), pad = (1024u - (raw & 1023u)) & 1023u;
    uint8_t *const shared = shared_raw + pad;
    uint4 *const queries = reinterpret_cast<uint4 *>(shared + S::kRing + S::kScales + S::kBars);  // left operands: [MMA][lane]
    float *const join = reinterpret_cast<float *>(queries) + S::kQueries / 4;
    float *const small = join + S::kJoin / 4;
    float *const tops = small, *const sums = small + kWarps * kAttentionRows;  // [warp][row]
    float *const row_scales = small + 2 * kWarps * kAttentionRows;             // [row] scale of the scores, in powers of two
    uint64_t *const scratch = reinterpret_cast<uint64_t *>(row_scales + kAttentionRows);
    uint32_t *const arrived = reinterpret_cast<uint32_t *>(scratch + 3 * kWarps + 2);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, row = lane >> 2, quad = lane & 3u;
    const uint32_t ring = raw + pad + warp * S::kSlots * S::kSlot, scales = raw + pad + S::kRing + warp * S::kSlots * S::kSlotScales;
    const uint32_t bars = raw + pad + S::kRing + S::kScales + warp * S::kSlots * 8, queries_at = raw + pad + S::kRing + S::kScales + S::kBars + lane * 16;
    if (lane == 0)
        for (uint32_t i = 0; i < S::kSlots; ++i) mbar_init(bars + i * 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    grid_dependency_wait();
    grid_dependents_launch();

    const Share share = share_of_block(p, g, scratch);
    if (share.any) {
        Asker<FMT, HDP> asker;
        asker.start(share, p, g, warp, lane);
        for (uint32_t i = 0; i < S::kSlots; ++i) asker.ask(p, g, &k_map, &v_map, ring, scales, bars, warp, lane);
        uint32_t slot = 0, parity = 0;
        unsigned long long limit_ns = kWaitLimitNs;
        Cursor at = share.at;
        do {
            // ---- queries of the item: warp w brings row w, split into halves, in the order in which key rows are read ----
            const uint32_t head = at.item / g.chunks, chunk = at.item % g.chunks;
            {
                const uint32_t r = chunk * kAttentionRows + warp, d = lane * 8;
                float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (r < g.rows && d < p.kv.head_dim) {
                    const uint64_t base = ((uint64_t)at.s * p.q_tokens + r / g.group) * p.q_stride + ((uint64_t)head * g.group + r % g.group) * p.kv.head_dim + d;
                    if (p.q_is_f32) {
                        const float4 *f = reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + base);
                        const float4 v = __ldcg(f), w = __ldcg(f + 1);
                        q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w, q[4] = w.x, q[5] = w.y, q[6] = w.z, q[7] = w.w;
                    } else {
                        const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + base));
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) q[2 * i] = __uint_as_float(w[i] << 16), q[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                    }
                }
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
                    const uint32_t m = (seg * S::kPieces + in_seg % S::kPieces) * kPer + d % S::kChunkDims / 4, to = warp * 4 + in_seg / S::kPieces;
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
                    queries[m * 32 + to] = a;
                    queries[(m + 1) * 32 + to] = b;
                }
                if (lane == 0) row_scales[warp] = row_scale;
            }
            __syncthreads();
            const float row_scale = row_scales[row];
            // tokens of the segment that all rows see, that this row sees, and that exist
            const int32_t end_token = (int32_t)(at.end * kTileTokens), existing = min(at.length, end_token);
            const int32_t sure = min(at.length - (int32_t)p.q_tokens + 1, end_token);
            const uint32_t r = chunk * kAttentionRows + row;
            const int32_t limit = r < g.rows ? min(at.length - (int32_t)p.q_tokens + 1 + (int32_t)(r / g.group), end_token) : 0;
            float acc[S::kAcc][4];
#pragma unroll
            for (uint32_t i = 0; i < S::kAcc; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            float top = kNone, sum = 0.f;                     // reference of the row's scores; sum of this lane's weights
            float weight_top = kNone, lift = 0.f, most = 0.f;  // 8-bit: reference of weights times scales, 2^(top - weight_top), and what they may be

            for (uint32_t tile = at.begin + warp * kStep; tile < at.end; tile += kWarps * kStep) {
                const int32_t token = (int32_t)(tile * kTileTokens);
                const bool edge = token + (int32_t)(kStep * kTileTokens) > sure;  // some rows do not see all of it
                // ---- scores ----
                mbar_wait(bars + slot * 8, parity, limit_ns, p.error_flag);
                float x[4 * kStep];  // this lane's: tokens 2 quad, + 1, + 8, + 9 of each tile, row `row`
                {
                    const uint32_t keys = ring + slot * S::kSlot;
                    float s[2 * kStep][4];
                    int upper[2 * kStep][4], lower[2 * kStep][4];  // int8: products with digits 3 and 2, and with 1 and 0
#pragma unroll
                    for (uint32_t n = 0; n < 2 * kStep; ++n) {
                        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                        upper[n][0] = upper[n][1] = upper[n][2] = upper[n][3] = lower[n][0] = lower[n][1] = lower[n][2] = lower[n][3] = 0;
                    }
#pragma unroll
                    for (uint32_t seg = 0; seg < S::kSegs; ++seg)
#pragma unroll
                        for (uint32_t c = 0; c < S::kPieces; ++c) {
                            const uint32_t piece = quad * S::kPieces + c, turn = S::kSeg == 128 ? row : row >> 1 & 3u;
                            const uint32_t within = seg * (kTileTokens * S::kSeg) + row * S::kSeg + ((piece ^ turn) << 4);
                            constexpr uint32_t kPer = S::kChunkDims / 4;
                            const uint32_t m = (seg * S::kPieces + c) * kPer;
                            uint32_t word[2 * kStep][4];
#pragma unroll
                            for (uint32_t n = 0; n < 2 * kStep; ++n) {
                                const uint4 w = lds_v4(keys + n / 2 * S::kTile + within + n % 2 * 8 * S::kSeg);
                                word[n][0] = w.x, word[n][1] = w.y, word[n][2] = w.z, word[n][3] = w.w;
                            }
#pragma unroll
                            for (uint32_t i = 0; i < kPer; ++i) {
                                const uint4 w = lds_v4(queries_at + (m + i) * 512);
                                const uint32_t qa[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (uint32_t n = 0; n < 2 * kStep; ++n) {
                                    if (FMT == 0) mma<FMT>(s[n], qa, word[n][2 * i], word[n][2 * i + 1]);
                                    else if (FMT == 1) mma_s8s8_16832(i % 2 == 0 ? upper[n] : lower[n], qa[0], qa[1], qa[2], qa[3], word[n][i / 2 * 2], word[n][i / 2 * 2 + 1]);
                                    else mma<FMT>(s[n], qa, e4m3_pair(word[n][i]), e4m3_pair(word[n][i] >> 16));
                                }
                            }
                        }
#pragma unroll
                    for (uint32_t n = 0; n < 2 * kStep; ++n) {
                        if (FMT == 1) {
                            // a sum of 256 products is below 2^22, so two digits' sums fit 32 bits
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                x[2 * n + j] = fmaf((float)(upper[n][j] * 256 + upper[n][j + 2]), 65536.f, (float)(lower[n][j] * 256 + lower[n][j + 2])) * row_scale;
                        } else {
                            x[2 * n] = (s[n][0] + s[n][2]) * row_scale;
                            x[2 * n + 1] = (s[n][1] + s[n][3]) * row_scale;
                        }
                        if (FMT != 0) {
                            const uint2 k = lds_v2(scales + slot * S::kSlotScales + n * 32 + quad * 8);
                            x[2 * n] *= __uint_as_float(k.x), x[2 * n + 1] *= __uint_as_float(k.y);
                        }
                    }
                }
                __syncwarp();  // the slot has been read
                asker.ask(p, g, &k_map, &v_map, ring, scales, bars, warp, lane);
                slot = slot + 1 == S::kSlots ? 0 : slot + 1;
                parity ^= slot == 0;
                if (edge)
#pragma unroll
                    for (uint32_t i = 0; i < 4 * kStep; ++i)
                        if (token + (int32_t)(i / 2 * 8 + quad * 2 + i % 2) >= limit) x[i] = -INFINITY;
                // ---- weights ----
                mbar_wait(bars + slot * 8, parity, limit_ns, p.error_flag);
                const uint32_t held = ring + slot * S::kSlot;
                float value_scale[FMT == 0 ? 1 : 4 * kStep], weight[4 * kStep];
                if (FMT != 0)
#pragma unroll
                    for (uint32_t n = 0; n < 2 * kStep; ++n) {
                        const uint2 v = lds_v2(scales + slot * S::kSlotScales + n * 32 + quad * 8);
                        value_scale[2 * n] = __uint_as_float(v.x), value_scale[2 * n + 1] = __uint_as_float(v.y);
                        // (a token that the row does not see: its scale may be anything)
                        if (edge) {
                            if (x[2 * n] == -INFINITY) value_scale[2 * n] = 0.f;
                            if (x[2 * n + 1] == -INFINITY) value_scale[2 * n + 1] = 0.f;
                        }
                    }
                float high = x[0], weight_high = 0.f;
#pragma unroll
                for (uint32_t i = 1; i < 4 * kStep; ++i) high = fmaxf(high, x[i]);
#pragma unroll
                for (uint32_t i = 0; i < 4 * kStep; ++i) {
                    weight[i] = exp2_fast(x[i] - top);
                    if (FMT != 0) weight_high = fmaxf(weight_high, weight[i] * value_scale[i]);
                }
                if (__any_sync(0xffffffffu, high - top > kHeadroom || (FMT != 0 && weight_high > most))) {
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
                    float keep = 1.f;
                    if (high - top > kHeadroom) {
                        high = ceilf(high);
                        keep = exp2_fast(top - high);
                        sum *= keep;
                        top = high;
                        if (FMT != 0) {
                            lift = weight_top == kNone ? 0.f : exp2_fast(top - weight_top);
                            most = lift > 0.f ? kMostWeight / lift : 0.f;
                            keep = 1.f;
                        }
#pragma unroll
                        for (uint32_t i = 0; i < 4 * kStep; ++i) weight[i] = exp2_fast(x[i] - top);
                    }
                    if (FMT != 0) {
                        weight_high = 0.f;
#pragma unroll
                        for (uint32_t i = 0; i < 4 * kStep; ++i) weight_high = fmaxf(weight_high, weight[i] * value_scale[i]);
                        weight_high = fmaxf(weight_high, __shfl_xor_sync(0xffffffffu, weight_high, 1));
                        weight_high = fmaxf(weight_high, __shfl_xor_sync(0xffffffffu, weight_high, 2));
                        if (weight_high > most) {
                            const int e = (int)(__float_as_uint(weight_high) >> 23) - 126;  // weight_high < 2^e
                            const float next = top + (float)max(e - kWeightExponent, -126);
                            keep = weight_top == kNone ? 0.f : exp2_fast(weight_top - next);
                            weight_top = next;
                            lift = exp2_fast(top - weight_top);
                            most = kMostWeight / lift;
                        }
                    }
#pragma unroll
                    for (uint32_t i = 0; i < S::kAcc; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] *= keep;
                }
#pragma unroll
                for (uint32_t i = 0; i < 4 * kStep; ++i) {
                    if (FMT != 0) {
                        sum += weight[i];
                        weight[i] *= value_scale[i] * lift;
                    }
                }
                uint32_t pa[kStep][4];
#pragma unroll
                for (uint32_t i = 0; i < kStep; ++i) {
                    split<FMT>(weight[4 * i], weight[4 * i + 1], pa[i][0], pa[i][1]);
                    split<FMT>(weight[4 * i + 2], weight[4 * i + 3], pa[i][2], pa[i][3]);
                    // bf16: the weights as they are multiplied, so that they add up to one whatever the halves cut off
                    if (FMT == 0)
#pragma unroll
                        for (int j = 0; j < 4; j += 2)
                            sum += (__uint_as_float(pa[i][j] << 16) + __uint_as_float(pa[i][j + 1] << 16)) +
                                   (__uint_as_float(pa[i][j] & 0xffff0000u) + __uint_as_float(pa[i][j + 1] & 0xffff0000u));
                }
                // ---- values ----
                if (edge) {
                    // Rows behind the sequence's end hold anything: zeros are put in their place. Among draft tokens a value that is not
                    // finite may be seen by some rows only, and a weight of zero does not take it out of a sum: it is added here to the
                    // rows that see it, and becomes a zero too.
#pragma unroll
                    for (uint32_t i = 0; i < kStep; ++i) {
                        const uint32_t base = held + i * S::kTile;
                        const int32_t first = token + (int32_t)(i * kTileTokens);
                        if (FMT != 1 && p.q_tokens > 1) {
                            bool odd = false;
                            for (uint32_t b = lane * 16; b < S::kTile; b += 512) {
                                const uint4 w = lds_v4(base + b);
                                const uint32_t word[4] = {w.x, w.y, w.z, w.w};
                                if (first + (int32_t)(b / S::kSeg % kTileTokens) < existing)
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
#pragma unroll
                                        for (int k = 0; k < 4; k += FMT == 0 ? 2 : 1) odd = odd || not_finite<FMT>(word[j], k);
                            }
                            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                                for (uint32_t c = 0; c < S::kAcc; ++c)
#pragma unroll
                                    for (uint32_t j = 0; j < 2; ++j) {
                                        const uint32_t d = FMT == 0 ? c * 8 + quad * 2 + j : c / 2 * 16 + quad * 4 + j * 2 + (c & 1u);
                                        const uint32_t byte = d * (FMT == 0 ? 2 : 1), seg = byte / S::kSeg, piece = byte % S::kSeg / 16;
                                        for (int32_t t = 0; t < (int32_t)kTileTokens && first + t < limit; ++t) {
                                            const uint32_t swap = S::kSeg == 128 ? (uint32_t)t & 7u : (uint32_t)t >> 1 & 3u;
                                            const uint32_t w = lds_u32((base + seg * (kTileTokens * S::kSeg) + (uint32_t)t * S::kSeg + ((piece ^ swap) << 4) + byte % 16) & ~3u);
                                            if (not_finite<FMT>(w, byte & 3u)) acc[c][j] += FMT == 0 ? __uint_as_float((w >> ((byte & 3u) * 8)) << 16) : __uint_as_float(0x7fc00000u);
                                        }
                                    }
                                __syncwarp();
                                for (uint32_t b = lane * 16; b < S::kTile; b += 512) {
                                    const uint4 w = lds_v4(base + b);
                                    uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
#pragma unroll
                                        for (int k = 0; k < 4; k += FMT == 0 ? 2 : 1)
                                            if (not_finite<FMT>(word[j], k)) word[j] &= ~((FMT == 0 ? 0xffffu : 0xffu) << (k * 8));
                                    sts_v4(base + b, make_uint4(word[0], word[1], word[2], word[3]));
                                }
                            }
                        }
                        for (uint32_t b = lane * 16; b < S::kTile; b += 512)
                            if (first + (int32_t)(b / S::kSeg % kTileTokens) >= existing) sts_v4(base + b, make_uint4(0u, 0u, 0u, 0u));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into these slots
                    __syncwarp();
                }
                const uint32_t matrix = lane >> 3, line = (lane & 7u) + (matrix & 1u) * 8, turn = S::kSeg == 128 ? line & 7u : line >> 1 & 3u;
#pragma unroll
                for (uint32_t c = 0; c < S::kChunks; c += 2) {
                    const uint32_t seg = c / (S::kSeg / 16), piece = c % (S::kSeg / 16) + (matrix >> 1);
                    const uint32_t within = seg * (kTileTokens * S::kSeg) + line * S::kSeg + ((piece ^ turn) << 4);
#pragma unroll
                    for (uint32_t t = 0; t < kStep; ++t) {
                        uint32_t v[4];
                        ldmatrix_x4_trans(v, held + t * S::kTile + within);
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i) {
                            const uint32_t b0 = v[2 * i], b1 = v[2 * i + 1];
                            if (FMT == 0) {
                                mma<FMT>(acc[c + i], pa[t], b0, b1);
                            } else if (FMT == 1) {
                                mma<FMT>(acc[(c + i) * 2], pa[t], int8_even(b0), int8_even(b1));
                                mma<FMT>(acc[(c + i) * 2 + 1], pa[t], int8_even(b0 >> 8), int8_even(b1 >> 8));
                            } else {
                                mma<FMT>(acc[(c + i) * 2], pa[t], e4m3_pair(__byte_perm(b0, 0, 0x4420)), e4m3_pair(__byte_perm(b1, 0, 0x4420)));
                                mma<FMT>(acc[(c + i) * 2 + 1], pa[t], e4m3_pair(__byte_perm(b0, 0, 0x4431)), e4m3_pair(__byte_perm(b1, 0, 0x4431)));
                            }
                        }
                    }
                }
                __syncwarp();
                asker.ask(p, g, &k_map, &v_map, ring, scales, bars, warp, lane);
                slot = slot + 1 == S::kSlots ? 0 : slot + 1;
                parity ^= slot == 0;
            }

            // ---- join the warps' results; then, in the last block of a cut item, those of the blocks ----
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            // what of the row's result a lane holds: dimensions 16 i + 4 quad ... + 3 (bf16, at first: 16 i + 2 quad, + 1, + 8, + 9)
            float4 o[HDP / 16];
#pragma unroll
            for (uint32_t i = 0; i < HDP / 16; ++i) {
                const float *a = acc[2 * i], *b = acc[2 * i + 1];
                o[i] = FMT == 0 ? make_float4(a[0] + a[2], a[1] + a[3], b[0] + b[2], b[1] + b[3]) : make_float4(a[0] + a[2], b[0] + b[2], a[1] + a[3], b[1] + b[3]);
            }
            if (top == kNone) top = -INFINITY;
            float o_top = FMT == 0 ? top : weight_top == kNone ? -INFINITY : weight_top;
            const bool cut = !at.whole_item();
            uint32_t owner, contributors;
            at.contributors(share.cut, blockIdx.x, &owner, &contributors);
            // a partial result: rows, then maxima, then sums
            constexpr uint32_t kPart = kAttentionRows * (kMaxHeadDim + 2);
            float *const part = p.parts + ((uint64_t)blockIdx.x * 2 + (blockIdx.x == owner ? 1 : 0)) * kPart;
            const uint32_t jr = threadIdx.x >> 4 & 7u, jd = (threadIdx.x & 15u) * 4;  // row and dimensions that a thread joins
            const uint32_t j_row = chunk * kAttentionRows + jr, j_draft = j_row / g.group;
            const bool j_live = j_row < g.rows, j_empty = at.length - (int32_t)p.q_tokens + 1 + (int32_t)j_draft <= 0;
            const uint64_t out_row = ((uint64_t)at.s * p.q_tokens + j_draft) * p.out_stride + ((uint64_t)head * g.group + j_row % g.group) * p.kv.head_dim;
            bool partial = cut;
            while (true) {
                if (quad == 0) {
                    tops[warp * kAttentionRows + row] = top;
                    sums[warp * kAttentionRows + row] = sum;
                }
                __syncthreads();
                float all_top = -INFINITY;
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) all_top = fmaxf(all_top, tops[w * kAttentionRows + row]);
                // (a warp without tiles, and rows that see nothing, have zeros; a row whose scores are NaNs keeps those)
                const float factor = o_top == -INFINITY ? 0.f : exp2_fast(o_top - all_top);
                float row_top = -INFINITY, total = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) row_top = fmaxf(row_top, tops[w * kAttentionRows + jr]);
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) {
                    const float t = tops[w * kAttentionRows + jr];
                    total += sums[w * kAttentionRows + jr] * (t == -INFINITY ? 1.f : exp2_fast(t - row_top));
                }
                const float by = 1.f / total;
#pragma unroll
                for (uint32_t round = 0; round < HDP / kRoundDims; ++round) {
                    float *const mine = join + (warp * kAttentionRows + row) * kRoundPitch;
#pragma unroll
                    for (uint32_t i = 0; i < kRoundDims / 16; ++i) {
                        float4 v = o[round * (kRoundDims / 16) + i];
                        v.x *= factor, v.y *= factor, v.z *= factor, v.w *= factor;
                        if (FMT == 0 && partial == cut) {
                            *reinterpret_cast<float2 *>(mine + i * 16 + quad * 2) = make_float2(v.x, v.y);
                            *reinterpret_cast<float2 *>(mine + i * 16 + 8 + quad * 2) = make_float2(v.z, v.w);
                        } else {
                            *reinterpret_cast<float4 *>(mine + i * 16 + quad * 4) = v;
                        }
                    }
                    __syncthreads();
                    if (threadIdx.x < 128) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (uint32_t w = 0; w < kWarps; ++w) {
                            const float4 a = *reinterpret_cast<const float4 *>(join + (w * kAttentionRows + jr) * kRoundPitch + jd);
                            v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
                        }
                        const uint32_t d = round * kRoundDims + jd;
                        if (partial) {
                            if (j_live) *reinterpret_cast<float4 *>(part + jr * HDP + d) = v;
                            if (round == 0 && jd == 0) {
                                part[kAttentionRows * HDP + jr] = row_top;
                                part[kAttentionRows * (HDP + 1) + jr] = total;
                            }
                        } else if (j_live && d < p.kv.head_dim) {
                            v = j_empty ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
                            if (p.out_is_f32) *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + out_row + d) = v;
                            else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + out_row + d) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                        }
                    }
                    if (round + 1 < HDP / kRoundDims) __syncthreads();
                }
                if (partial) __threadfence();
                __syncthreads();
                if (!partial) break;
                if (threadIdx.x == 0) {
                    *arrived = atomicAdd(p.counters + owner, 1u) + 1 == contributors;
                    if (*arrived) p.counters[owner] = 0;
                    __threadfence();
                }
                __syncthreads();
                if (!*arrived) break;
                // partial results in the order of the tiles: warp w adds up those of blocks w, w + 8, ...
                partial = false;
                const float *const parts = p.parts + (uint64_t)owner * 2 * kPart;
                auto part_of = [&](uint32_t i) { return parts + (i * 2 + (i == 0 ? 1 : 0)) * kPart; };
                top = -INFINITY;
                sum = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < HDP / 16; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (uint32_t i = warp; i < contributors; i += kWarps) top = fmaxf(top, __ldcg(part_of(i) + kAttentionRows * HDP + row));
                o_top = top;
                for (uint32_t i = warp; i < contributors; i += kWarps) {
                    const float *const from = part_of(i);
                    const float t = __ldcg(from + kAttentionRows * HDP + row), l = __ldcg(from + kAttentionRows * (HDP + 1) + row);
                    float4 v[HDP / 16];
                    if (chunk * kAttentionRows + row < g.rows) {
#pragma unroll
                        for (uint32_t j = 0; j < HDP / 16; ++j) v[j] = __ldcg(reinterpret_cast<const float4 *>(from + row * HDP + j * 16 + quad * 4));
                        const float f = t == -INFINITY ? 0.f : exp2_fast(t - top);
                        sum += t == -INFINITY ? l : l * f;
#pragma unroll
                        for (uint32_t j = 0; j < HDP / 16; ++j)
                            o[j].x = fmaf(v[j].x, f, o[j].x), o[j].y = fmaf(v[j].y, f, o[j].y), o[j].z = fmaf(v[j].z, f, o[j].z), o[j].w = fmaf(v[j].w, f, o[j].w);
                    }
                }
            }
        } while (at.next([&](uint32_t i) { return length_of(p, i); }, p.kv.sequences, g.heads));
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

// Rows of the cache as [page][head][token][value]; copies of 16 tokens by one segment.
template <int FMT, int HDP>
bool encode_map(EncodeTiledFn encode, CUtensorMap *map, const KvView &kv, const uint8_t *pool) {
    using S = Shape<FMT, HDP>;
    const cuuint64_t dims[4] = {kv.head_dim, kv.page_tokens, kv.kv_heads, kv.pages};
    const cuuint64_t strides[3] = {kv.token_stride, kv.head_stride, kv.page_stride};
    const cuuint32_t box[4] = {S::kSeg / (FMT == 0 ? 2 : 1), kTileTokens, 1, 1}, step[4] = {1, 1, 1, 1};
    return encode(map, FMT == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t *>(pool), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, S::kSeg == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, int HDP>
cudaError_t launch(const AttentionParams &p, uint32_t sm_count, cudaStream_t stream) {
    using S = Shape<FMT, HDP>;
    const EncodeTiledFn encode = encode_tiled_fn();
    CUtensorMap maps[2];
    if (!encode || !encode_map<FMT, HDP>(encode, &maps[0], p.kv, p.kv.k) || !encode_map<FMT, HDP>(encode, &maps[1], p.kv, p.kv.v)) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> ready{0};  // a bit for each device: the attribute is the kernel's, once set it stays
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(attention_kernel<FMT, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kShared);
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    Geometry g;
    g.group = p.heads / p.kv.kv_heads;
    g.rows = g.group * p.q_tokens;
    g.chunks = (g.rows + kAttentionRows - 1) / kAttentionRows;
    g.heads = p.kv.kv_heads * g.chunks;
    g.pages = attention_pages(p.kv.page_tokens);
    return launch_dependent(attention_kernel<FMT, HDP>, dim3(sm_count), kThreads, S::kShared, stream, p, g, maps[0], maps[1]);
}

template <int FMT>
cudaError_t launch_dim(const AttentionParams &p, uint32_t sm_count, cudaStream_t stream) {
    if (p.kv.head_dim <= 64) return launch<FMT, 64>(p, sm_count, stream);
    if (p.kv.head_dim <= 128) return launch<FMT, 128>(p, sm_count, stream);
    return launch<FMT, 256>(p, sm_count, stream);
}

}  // namespace q4

extern "C" size_t q4k_attention_part_floats(uint32_t sm_count) { return (size_t)sm_count * 2 * q4::kAttentionRows * (q4::kMaxHeadDim + 2); }

extern "C" cudaError_t q4k_attention(const q4::AttentionParams *p, uint32_t sm_count, cudaStream_t stream) {
    if (p->kv.format == 0u) return q4::launch_dim<0>(*p, sm_count, stream);
    if (p->kv.format == 1u) return q4::launch_dim<1>(*p, sm_count, stream);
    return q4::launch_dim<2>(*p, sm_count, stream);
}
