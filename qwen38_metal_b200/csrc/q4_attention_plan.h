// How the work of an attention call is cut over its blocks; shared by the kernel and the CPU tests.
//
// A tile is 16 tokens of one sequence, which lie in one page. An item is what one result belongs to: a sequence, a key head and eight
// query rows of it; it has as many tiles as its sequence. Blocks take runs of tiles, and the partial results of an item that
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
constexpr uint32_t kAttentionRows = 8;  // query rows of an item

Q4_PLAN_FN uint32_t attention_tiles(int64_t length) { return length > 0 ? (uint32_t)((length + kTileTokens - 1) / kTileTokens) : 0u; }

// The cut of a call, the same in every block.
struct AttentionCut {
    uint64_t run;      // tiles of a block's share, or of a piece at most
    uint32_t whole;    // 1: every block takes one piece of one item; 0: blocks take equal runs through all tiles
};

// `tiles`: of all items; `items`: those that have any. With few items every item is cut into equal pieces, one to a block: no block
// has a second start or an uneven rest. pieces <= tiles / run + items <= blocks holds for run >= tiles / (blocks - items).
Q4_PLAN_FN AttentionCut attention_cut(uint64_t tiles, uint64_t items, uint32_t blocks, uint32_t least) {
    AttentionCut c;
    c.whole = items * 2 <= blocks ? 1u : 0u;
    const uint64_t by = c.whole ? blocks - items : blocks;
    c.run = (tiles + by - 1) / by;
    if (c.run < least) c.run = least;
    return c;
}

Q4_PLAN_FN uint64_t attention_pieces(const AttentionCut &c, uint32_t tiles) { return (tiles + c.run - 1) / c.run; }

// What a sequence counts for in the search for a block's start: its pieces, or its tiles, in all items.
Q4_PLAN_FN uint64_t attention_weight(const AttentionCut &c, uint32_t tiles, uint32_t items) {
    return (c.whole ? attention_pieces(c, tiles) : (uint64_t)tiles) * items;
}

// Walks the segments of a block's share: tiles [begin, end) of an item. `items` of a sequence, `lengths(s)` its tokens.
struct AttentionCursor {
    uint32_t s, item, begin, end, tiles;
    uint32_t piece, pieces;  // of an item cut into equal pieces
    int32_t length;
    uint64_t left;   // tiles of the share from `begin` on
    uint64_t first;  // equal runs: number of the sequence's first tile among the tiles of all items

    Q4_PLAN_FN void close() { end = (uint64_t)(tiles - begin) < left ? tiles : begin + (uint32_t)left; }

    // Start of the block's share, which begins `local` pieces or tiles into sequence s; `before`: those of the sequences in front.
    Q4_PLAN_FN void start(const AttentionCut &cut, uint32_t sequence, int64_t tokens, uint64_t before, uint64_t local, uint64_t all_tiles) {
        s = sequence;
        length = (int32_t)tokens;
        tiles = attention_tiles(tokens);
        first = before;
        piece = 0;
        pieces = 1;
        if (cut.whole) {
            pieces = (uint32_t)attention_pieces(cut, tiles);
            item = (uint32_t)(local / pieces);
            piece = (uint32_t)(local % pieces);
            begin = (uint32_t)((uint64_t)tiles * piece / pieces);
            left = (uint32_t)((uint64_t)tiles * (piece + 1) / pieces) - begin;
        } else {
            item = (uint32_t)(local / tiles);
            begin = (uint32_t)(local % tiles);
            left = all_tiles - (before + local) < cut.run ? all_tiles - (before + local) : cut.run;
        }
        close();
    }

    template <typename Lengths>
    Q4_PLAN_FN bool next(const Lengths &lengths, uint32_t sequences, uint32_t items) {
        left -= end - begin;
        if (left == 0) return false;
        begin = 0;
        if (++item == items) {
            item = 0;
            first += (uint64_t)tiles * items;
            do {
                if (++s >= sequences) return false;  // (never: `left` counts tiles that exist)
                const int64_t tokens = lengths(s);
                length = (int32_t)tokens;
                tiles = attention_tiles(tokens);
            } while (tiles == 0);
        }
        close();
        return true;
    }

    Q4_PLAN_FN bool whole_item() const { return begin == 0 && end == tiles; }

    // Blocks owner ... owner + contributors - 1 work on the item. A block is the owner of one cut item at most, its share's last
    // one, and one of the others of one at most, its first: two places for partial results are enough, place 1 for an owner.
    Q4_PLAN_FN void contributors(const AttentionCut &cut, uint32_t block, uint32_t *owner, uint32_t *count) const {
        if (cut.whole) {
            *owner = block - piece;
            *count = pieces;
            return;
        }
        const uint64_t from = first + (uint64_t)item * tiles;
        *owner = (uint32_t)(from / cut.run);
        *count = (uint32_t)((from + tiles - 1) / cut.run) - *owner + 1;
    }
};

}  // namespace q4
