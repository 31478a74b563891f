// Host build of index arithmetic of the attention operators (qwen38_metal_b200/csrc/q4_attention_plan.h) for CPU tests.
#include "../qwen38_metal_b200/csrc/q4_attention_plan.h"
extern "C" {
uint64_t shim_kv_scale_index(uint64_t first, uint32_t head, uint32_t page_tokens) { return q4::kv_scale_index(first, head, page_tokens); }
int shim_attention_hidden(int32_t token, int32_t tokens, int32_t sure) { return q4::attention_some_hidden(token, tokens, sure); }
}
