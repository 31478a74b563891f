// How the work of an attention call is cut over its blocks; shared by the kernel and the CPU tests.
//
// A tile is 16 tokens of one sequence, or 16 << shift where pages have a whole number of those: tokens that lie in one page and come by
// one copy. An item is what one result belongs to: a sequence, a key head and 8, 16 or 24 query rows of it; it has as many tiles as its
// sequence. Blocks take runs of tiles, and the partial results of an item that
// several blocks have worked on are joined by the last of them.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define Q4_PLAN_FN __host__ __device__ __forceinline__
#else
#define Q4_PLAN_FN inline
#endif

namespace q4 {

constexpr uint32_t kTileTokens = 16;
constexpr uint32_t kAttentionRows = 8;  // query rows that are multiplied together

// Scales lie [page][key head][token of the page]: number of a head's, `first` being that of head 0. Heads times tokens may pass 32 bits.
Q4_PLAN_FN uint64_t kv_scale_index(uint64_t first, uint32_t head, uint32_t page_tokens) { return first + (uint64_t)head * page_tokens; }

Q4_PLAN_FN uint32_t attention_tiles(int64_t length, uint32_t shift) { return length > 0 ? (uint32_t)((length - 1) / kTileTokens >> shift) + 1 : 0u; }

// tile / per for tiles below 2^27, as a product: 2^(32 + shift) / per rounded up is off by less than per <= 2^(shift + 1).
struct AttentionPages {
    uint32_t per, inverse, shift;  // tiles of a page
    Q4_PLAN_FN uint32_t page_of(uint32_t tile) const { return per == 1 ? tile : (uint32_t)((uint64_t)tile * inverse >> 32) >> shift; }
};
inline AttentionPages attention_pages(uint32_t page_tokens, uint32_t tile_shift) {
    AttentionPages d = {page_tokens / (kTileTokens << tile_shift), 0, 0};
    while ((2ull << d.shift) < d.per) ++d.shift;
    if (d.per > 1) d.inverse = (uint32_t)(((1ull << (32 + d.shift)) + d.per - 1) / d.per);
    return d;
}

// Whether some rows do not see all of `tokens` tokens from `token` on, the first `sure` ones being seen by all. (The last token's number plus one
// step may pass 31 bits.)
Q4_PLAN_FN bool attention_some_hidden(int32_t token, int32_t tokens, int32_t sure) { return token > sure - tokens; }

enum AttentionMode : uint32_t {
    kEqualRuns = 0,    // blocks take equal runs through the tiles of all items
    kEqualPieces = 1,  // every item is cut into equal pieces, a block takes one
    kWholeItems = 2    // blocks take the items whose middle lies in their run
};

// The cut of a call, the same in every block. All numbers of tiles fit 32 bits: the host refuses calls that could have more.
struct AttentionCut {
    uint32_t tiles;  // of all items
    uint32_t run;    // tiles of a block's run, or of a piece at most
    uint32_t mode;
    uint32_t shift;  // of a tile's tokens
};

// `tiles`: of all items, `items`: those that have any, `longest`: tiles of the longest one.
//   * Items stay whole where that costs a block no more than four times `least` tiles: what joining cut items takes. Where each has a block of its
//     own a piece is as long as the longest; more of them go by where their middles lie. (Int8, 4 key heads of 256, whole against cut: 128 items of
//     800 / 1600 / 3600 tokens 22.5 / 32.8 / 57.3 us against 26.6 / 36.9 / 61.4; 52 items of 800 / 1600 / 3600 tokens 18.4 / 26.6 / 45.1 against
//     22.5 / 26.6 / 36.9; 240 items of 800 / 3600 tokens 38.9 / 104.4 against 43.0 / 102.4. Few items leave most blocks idle, and joining is all
//     that goes on: 4 items of 300 / 600 / 1000 tokens 14.3 / 16.4 / 18.4 against 16.3 / 16.4 / 16.4.)
//   * Few items are cut into pieces: no block has a second start or an uneven rest. pieces <= tiles / run + items <= blocks
//     holds for run >= tiles / (blocks - items). (Above a third of the blocks the longer runs cost more: 64 items 74 us, in equal runs 55 us.)
//   * Otherwise all blocks take the same number of tiles.
Q4_PLAN_FN AttentionCut attention_cut(uint32_t tiles, uint32_t items, uint32_t longest, uint32_t blocks, uint32_t least, uint32_t shift) {
    AttentionCut c;
    c.shift = shift;
    c.tiles = tiles;
    const uint32_t even = (tiles - 1) / blocks + 1, more = longest > even ? longest - even : 0;
    const bool few = items <= blocks / 3;
    if (items <= blocks && more <= (few ? 2 : 4) * least) {
        c.mode = kEqualPieces;
        c.run = longest;
    } else if (few) {
        c.mode = kEqualPieces;
        c.run = (tiles - 1) / (blocks - items) + 1;
        if (c.run < least) c.run = least;
    } else {
        c.mode = longest <= 4 * least || longest <= even / 16 ? kWholeItems : kEqualRuns;
        c.run = even < least && c.mode == kEqualRuns ? least : even;
    }
    return c;
}

Q4_PLAN_FN uint32_t attention_pieces(const AttentionCut &c, uint32_t tiles) { return tiles == 0 ? 0 : (tiles - 1) / c.run + 1; }

// What a sequence counts for in the search for a block's start: its pieces, or its tiles, in all items.
Q4_PLAN_FN uint32_t attention_weight(const AttentionCut &c, uint32_t tiles, uint32_t items) {
    return (c.mode == kEqualPieces ? attention_pieces(c, tiles) : tiles) * items;
}

// Where block `block` starts, in those. False: behind them, it has nothing to do.
Q4_PLAN_FN bool attention_target(const AttentionCut &c, uint32_t block, uint32_t *target) {
    const uint64_t to = c.mode == kEqualPieces ? block : (uint64_t)block * c.run;
    *target = (uint32_t)to;
    return c.mode == kEqualPieces || to < c.tiles;
}

// Walks the segments of a block's share: tiles [begin, end) of an item. `items` of a sequence, `lengths(s)` its tokens.
struct AttentionCursor {
    uint32_t s, item, begin, end, tiles;
    uint32_t piece, pieces;  // of an item cut into equal pieces
    int32_t length;
    uint32_t left;   // tiles of the share from `begin` on; whole items: where the block's run ends
    uint32_t first;  // runs: number of the sequence's first tile among the tiles of all items
    uint32_t whole, shift;

    Q4_PLAN_FN void close() { end = whole || tiles - begin < left ? tiles : begin + left; }
    Q4_PLAN_FN bool mine() const { return first + item * tiles + tiles / 2 < left; }  // whole items: middle in the run

    // Start of the block's share, which lies `target - before` pieces or tiles into sequence `sequence`; `before`: those of the
    // sequences in front. False: whole items, and none has its middle in the block's run.
    template <typename Lengths>
    Q4_PLAN_FN bool start(const AttentionCut &cut, uint32_t target, uint32_t sequence, uint32_t before, const Lengths &lengths, uint32_t sequences, uint32_t items) {
        const int64_t tokens = lengths(sequence);
        const uint32_t local = target - before;
        s = sequence;
        length = (int32_t)tokens;
        shift = cut.shift;
        tiles = attention_tiles(tokens, shift);
        first = before;
        piece = 0;
        pieces = 1;
        whole = cut.mode == kWholeItems;
        if (cut.mode == kEqualPieces) pieces = attention_pieces(cut, tiles);
        const uint32_t per = cut.mode == kEqualPieces ? pieces : tiles;
        item = local / per;
        begin = local - item * per;
        left = cut.tiles - target < cut.run ? cut.tiles - target : cut.run;
        bool behind = false;
        if (cut.mode == kEqualPieces) {
            // the first `longer` pieces have a tile more than the others
            const uint32_t each = tiles / pieces, longer = tiles - each * pieces;
            piece = begin;
            begin = piece * each + (piece < longer ? piece : longer);
            left = each + (piece < longer ? 1 : 0);
        } else if (whole) {
            left += target;
            behind = begin > tiles / 2;  // its middle lies in the run before
            begin = 0;
        }
        end = tiles;  // (next looks at it)
        if (behind) return next(lengths, sequences, items);
        if (whole && !mine()) return false;
        close();
        return true;
    }

    template <typename Lengths>
    Q4_PLAN_FN bool next(const Lengths &lengths, uint32_t sequences, uint32_t items) {
        if (!whole) {
            left -= end - begin;
            if (left == 0) return false;
        }
        begin = 0;
        if (++item == items) {
            item = 0;
            first += tiles * items;
            do {
                if (++s >= sequences) return false;
                const int64_t tokens = lengths(s);
                length = (int32_t)tokens;
                tiles = attention_tiles(tokens, shift);
            } while (tiles == 0);
        }
        if (whole && !mine()) return false;
        close();
        return true;
    }

    Q4_PLAN_FN bool whole_item() const { return begin == 0 && end == tiles; }

    // Blocks owner ... owner + contributors - 1 work on the item. A block is the owner of one cut item at most, its share's last
    // one, and one of the others of one at most, its first: two places for partial results are enough, place 1 for an owner.
    Q4_PLAN_FN void contributors(const AttentionCut &cut, uint32_t block, uint32_t *owner, uint32_t *count) const {
        *owner = block - piece;
        *count = pieces;
        if (cut.mode != kEqualRuns) return;
        const uint32_t from = first + item * tiles;
        *owner = from / cut.run;
        *count = (from + (tiles - 1)) / cut.run - *owner + 1;
    }
};

}  // namespace q4
