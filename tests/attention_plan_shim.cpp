// Host build of how attention cuts its work (qwen38_metal_b200/csrc/q4_attention_plan.h) for CPU tests.
#include "../qwen38_metal_b200/csrc/q4_attention_plan.h"
extern "C" {
// All blocks' segments, seven numbers each: block, sequence, item, begin, end, owner, contributors. Returns how many.
uint64_t shim_attention_plan(const int64_t *lengths, uint32_t sequences, uint32_t items, uint32_t blocks, uint32_t least, uint64_t *out, uint64_t most) {
    uint64_t tiles = 0, live = 0, n = 0;
    for (uint32_t s = 0; s < sequences; ++s) {
        tiles += q4::attention_tiles(lengths[s]);
        live += lengths[s] > 0;
    }
    if (tiles == 0) return 0;
    tiles *= items;
    const q4::AttentionCut cut = q4::attention_cut(tiles, live * items, blocks, least);
    for (uint32_t b = 0; b < blocks; ++b) {
        const uint64_t target = cut.whole ? b : b * cut.run;
        uint64_t before = 0;
        for (uint32_t s = 0; s < sequences; ++s) {
            const uint64_t weight = q4::attention_weight(cut, q4::attention_tiles(lengths[s]), items);
            if (target >= before && target < before + weight) {
                q4::AttentionCursor c;
                c.start(cut, s, lengths[s], before, target - before, tiles);
                do {
                    if (n == most) return n;
                    uint32_t owner, count;
                    c.contributors(cut, b, &owner, &count);
                    const uint64_t row[7] = {b, c.s, c.item, c.begin, c.end, owner, count};
                    for (int i = 0; i < 7; ++i) out[n * 7 + i] = row[i];
                    ++n;
                } while (c.next([&](uint32_t i) { return lengths[i]; }, sequences, items));
                break;
            }
            before += weight;
        }
    }
    return n;
}
}
