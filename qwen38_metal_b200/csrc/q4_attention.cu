// Attention of new tokens over a paged cache. Counterparts in the reference: the cache's scores and values kernels
// (src/metal_runtime.rs:8230-8798, shaders/qwen38.metal:4761-5323).
//
//     out = sum_j p_j v_j / sum_j p_j,   p_j = e^(scale q.k_j)
//
// The plain form: a block per query row, a warp per token at a time, one pass with the running maximum and sum of every warp,
// joined through shared memory. Everything in 32 bits.
#include "q4_attention.h"

#include <cuda_fp8.h>

#include "q4_device.cuh"

namespace q4 {

constexpr uint32_t kWarps = 8;

__device__ __forceinline__ void cache8(const uint8_t *row, uint32_t d, uint32_t format, float scale, float (&v)[8]) {
    if (format == 0u) {
        const uint4 a = __ldcg(reinterpret_cast<const uint4 *>(row + 2 * d));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
        return;
    }
    const uint2 a = __ldcg(reinterpret_cast<const uint2 *>(row + d));
    const uint32_t w[2] = {a.x, a.y};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t pair = (w[i / 4] >> (i % 4 * 8)) & 0xffffu;
        if (format == 1u) {
            v[i] = (float)(int8_t)(pair & 0xffu) * scale;
            v[i + 1] = (float)(int8_t)(pair >> 8) * scale;
        } else {
            const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3)));
            v[i] = f.x * scale;
            v[i + 1] = f.y * scale;
        }
    }
}

__global__ void __launch_bounds__(kWarps * 32) attention_kernel(const AttentionParams p) {
    __shared__ float part[kWarps][kMaxHeadDim], tops[kWarps], sums[kWarps];
    grid_dependency_wait();
    grid_dependents_launch();
    const KvView &kv = p.kv;
    const uint32_t row = blockIdx.x, head = blockIdx.y, s = row / p.q_tokens, i = row % p.q_tokens;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, d = lane * 8u;
    const uint32_t kv_head = head / (p.heads / kv.kv_heads);
    int64_t length = __ldcg(p.lengths + s);
    const int64_t most = (int64_t)kv.per_sequence * kv.page_tokens;
    if (length < 0 || length > most) {
        if (threadIdx.x == 0) *kv.input_error = 1;
        length = length < 0 ? 0 : most;
    }
    const int64_t seen = length - p.q_tokens + 1 + i;
    const bool has = d < kv.head_dim;
    float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint64_t at = row * p.q_stride + (uint64_t)head * kv.head_dim + d;
    if (has)
        for (int j = 0; j < 8; ++j)
            q[j] = p.q_is_f32 ? __ldcg(static_cast<const float *>(p.q) + at + j) : __uint_as_float((uint32_t)__ldcg(static_cast<const uint16_t *>(p.q) + at + j) << 16);
    float top = -INFINITY, sum = 0.f;
    for (int64_t t = warp; t < seen; t += kWarps) {
        const uint32_t entry = (uint32_t)t / kv.page_tokens, slot = (uint32_t)t % kv.page_tokens;
        const uint32_t page = (uint32_t)__ldcg(kv.table + (uint64_t)s * kv.row_stride + entry);
        const bool there = page < kv.pages;
        if (!there && lane == 0) *kv.input_error = 1;
        float k[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (there && has) {
            const uint64_t off = (uint64_t)page * kv.page_stride + (uint64_t)kv_head * kv.head_stride + (uint64_t)slot * kv.token_stride;
            const uint64_t sc = ((uint64_t)page * kv.kv_heads + kv_head) * kv.page_tokens + slot;
            cache8(kv.k + off, d, kv.format, kv.format ? __ldcg(kv.k_scales + sc) : 1.f, k);
            cache8(kv.v + off, d, kv.format, kv.format ? __ldcg(kv.v_scales + sc) : 1.f, v);
        }
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(q[j], k[j], dot);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
        dot *= p.scale;
        const float next = fmaxf(top, dot);
        const float keep = next == -INFINITY ? 1.f : expf(top - next), w = expf(dot - next);
        sum = sum * keep + w;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = o[j] * keep + w * v[j];
        top = next;
    }
    if (has)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[warp][d + j] = o[j];
    if (lane == 0) tops[warp] = top, sums[warp] = sum;
    __syncthreads();
    float all = -INFINITY, total = 0.f;
    for (uint32_t w = 0; w < kWarps; ++w) all = fmaxf(all, tops[w]);
    const float base = all == -INFINITY ? 0.f : all;
    for (uint32_t w = 0; w < kWarps; ++w) total += sums[w] * expf(tops[w] - base);
    for (uint32_t e = threadIdx.x; e < kv.head_dim; e += blockDim.x) {
        float r = 0.f;
        for (uint32_t w = 0; w < kWarps; ++w) r += part[w][e] * expf(tops[w] - base);
        r = seen > 0 ? r / total : 0.f;
        const uint64_t to = row * p.out_stride + (uint64_t)head * kv.head_dim + e;
        if (p.out_is_f32) static_cast<float *>(p.out)[to] = r;
        else static_cast<__nv_bfloat16 *>(p.out)[to] = __float2bfloat16_rn(r);
    }
}

}  // namespace q4

extern "C" cudaError_t q4k_attention(const q4::AttentionParams *p, uint32_t, cudaStream_t stream) {
    return q4::launch_dependent(q4::attention_kernel, dim3(p->kv.sequences * p->q_tokens, p->heads), q4::kWarps * 32, 0, stream, *p);
}
