// Host build of how attention cuts its work (qwen38_metal_b200/csrc/q4_attention_plan.h) for CPU tests.
#include "../qwen38_metal_b200/csrc/q4_attention_plan.h"
extern "C" {
// All blocks' segments, seven numbers each: block, sequence, item, begin, end, owner, contributors. Returns how many.
uint64_t shim_attention_plan(const int64_t *lengths, uint32_t sequences, uint32_t items, uint32_t blocks, uint32_t least, uint32_t shift, uint64_t *out, uint64_t most) {
    uint64_t tiles = 0, live = 0, n = 0;
    uint32_t longest = 0;
    for (uint32_t s = 0; s < sequences; ++s) {
        const uint32_t t = q4::attention_tiles(lengths[s], shift);
        tiles += t;
        live += t > 0;
        longest = t > longest ? t : longest;
    }
    if (tiles == 0) return 0;
    if (tiles * items > 0xffffffffull) return 0;
    const q4::AttentionCut cut = q4::attention_cut((uint32_t)(tiles * items), (uint32_t)live * items, longest, blocks, least, shift);
    auto length = [&](uint32_t i) { return lengths[i]; };
    for (uint32_t b = 0; b < blocks; ++b) {
        uint32_t target, before = 0;
        if (!q4::attention_target(cut, b, &target)) continue;
        for (uint32_t s = 0; s < sequences; ++s) {
            const uint32_t weight = q4::attention_weight(cut, q4::attention_tiles(lengths[s], shift), items);
            if (target >= before && target - before < weight) {
                q4::AttentionCursor c;
                if (!c.start(cut, target, s, before, length, sequences, items)) break;
                do {
                    if (n == most) return n;
                    uint32_t owner, count;
                    c.contributors(cut, b, &owner, &count);
                    const uint64_t row[7] = {b, c.s, c.item, c.begin, c.end, owner, count};
                    for (int i = 0; i < 7; ++i) out[n * 7 + i] = row[i];
                    ++n;
                } while (c.next(length, sequences, items));
                break;
            }
            before += weight;
        }
    }
    return n;
}
uint32_t shim_attention_page_of(uint32_t page_tokens, uint32_t shift, uint32_t tile) { return q4::attention_pages(page_tokens, shift).page_of(tile); }
}
