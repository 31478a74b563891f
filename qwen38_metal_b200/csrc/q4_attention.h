// Kernel-side parameter blocks and launchers of the attention operators (rotary positions, paged cache, attention), and what
// their C entry points (q4_attention_api.cpp) need of the runtime. Plain C structs.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

struct q4b_runtime;

namespace q4 {

// What the entry points outside q4_runtime.cu use of a runtime.
struct RuntimeView {
    std::recursive_mutex *mu;
    int device;
    int sm_count;
    int *error_flag;   // device word: a bounded wait ran out
    int *input_error;  // device word: an index in device memory was out of range
    float *attention_parts;
    unsigned int *attention_counters;
    uint64_t *launches;
};
RuntimeView runtime_view(q4b_runtime *rt);
int set_error(int status, const char *message);

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int device) {
        cudaGetDevice(&prev);
        if (prev != device) cudaSetDevice(device);
        else prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

constexpr uint32_t kMaxHeadDim = 256;

// Pair i of a rotary turns by positions * step[i] / 2^64 turns.
struct RotaryView {
    const uint64_t *step;  // device, [pairs]; null: no rotation
    uint32_t pairs;
    uint32_t interleaved;
    float factor;
};

struct KvView {
    uint8_t *k, *v;
    float *k_scales, *v_scales;
    uint64_t page_stride, head_stride, token_stride;  // bytes
    uint32_t format, kv_heads, head_dim, page_tokens, pages;
    const int32_t *table;
    uint32_t sequences, per_sequence;
    uint64_t row_stride;  // entries
    int *input_error;
};

struct RotaryParams {
    RotaryView rotary;
    const void *x;
    void *out;
    const int32_t *positions;
    uint64_t x_stride, out_stride;  // values
    uint64_t tokens;
    uint32_t heads, head_dim;
    uint32_t x_is_f32, out_is_f32;
};

struct KvTokensParams {
    KvView kv;
    RotaryView rotary;
    const int32_t *positions, *sequences;
    const void *k_in, *v_in;  // write
    void *k_out, *v_out;      // read
    uint64_t k_stride, v_stride;  // values
    uint64_t tokens;
    uint32_t run;  // sequences null: tokens of each sequence
    uint32_t is_f32;
};

struct AttentionParams {
    KvView kv;
    const int32_t *lengths;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;  // values
    uint32_t heads, q_tokens;
    uint32_t q_is_f32, out_is_f32;
    float scale;
    float *parts;
    unsigned int *counters;
    int *error_flag;
};

}  // namespace q4

extern "C" {
cudaError_t q4k_rotary(const q4::RotaryParams *p, uint32_t sm_count, cudaStream_t stream);
cudaError_t q4k_kv_write(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream);
cudaError_t q4k_kv_read(const q4::KvTokensParams *p, uint32_t sm_count, cudaStream_t stream);
size_t q4k_attention_part_floats(uint32_t sm_count);  // scratch of partial results; one counter a block, zero between launches
cudaError_t q4k_attention(const q4::AttentionParams *p, uint32_t sm_count, cudaStream_t stream);
}
