/*
 * q4b200 -- what stands between a layer's Q/K/V projections and its output projection: rotary positions, a paged cache of
 * keys and values that is quantised as it is written, and attention of new tokens over that cache.
 *
 * Counterparts in the reference: the rotary preparation and the int8 cache with a scale for each token and head
 * (src/metal_runtime.rs:5171-5475, 7298-7457, 8230-8798; shaders/qwen38.metal:4761-5323) and the logical page table
 * (src/paged_kv.rs:1-163).
 *
 * The conventions are those of the `_device` calls of q4b200.h: device pointers, work enqueued on the stream that is given,
 * no synchronisation, outputs untouched when a call returns an error, calls on one runtime ordered on the device (they share
 * its scratch; a captured graph may be replayed as long as the runtime, the rotary handles that its calls were given and the
 * caller's buffers live). None of the `_device` calls allocates.
 *
 * Activations are rows of a token: heads x head_dim values, heads behind each other, `stride` VALUES from one token to the
 * next. Types Q4B_F32 and Q4B_BF16. Addresses are multiples of 16 bytes and so are strides in bytes, else
 * Q4B_INVALID_ARGUMENT. head_dim is a multiple of 16 from 16 to 256, else Q4B_UNSUPPORTED. No tokens, heads or sequences is
 * Q4B_EMPTY_DIMENSION. An output may not share memory with an input or with the cache; rotary alone works in place.
 *
 * What only the device can see -- a sequence number, a position behind the page table's last entry, a page number outside the
 * cache, a length longer than the page table or negative -- never reads or writes outside the caller's buffers: the token is
 * left out (attention: pages outside the cache count as zeros, lengths are cut to what exists), and the next
 * q4b_device_status returns Q4B_TENSOR_OUT_OF_RANGE.
 */
#ifndef Q4B_ATTENTION_H
#define Q4B_ATTENTION_H

#include "q4b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions ---- */

typedef enum q4b_rotary_layout {
    Q4B_ROTARY_HALF = 0,        /* pair i is (x[i], x[i + rotary_dim / 2]) */
    Q4B_ROTARY_INTERLEAVED = 1  /* pair i is (x[2 i], x[2 i + 1]) */
} q4b_rotary_layout;

typedef enum q4b_rotary_scaling_kind {
    Q4B_ROTARY_UNSCALED = 0,
    Q4B_ROTARY_LINEAR = 1,  /* positions divided by `factor` */
    Q4B_ROTARY_NTK = 2,     /* base * factor^(rotary_dim / (rotary_dim - 2)) */
    Q4B_ROTARY_YARN = 3     /* pairs that turn more than fast_turns times in original_length tokens keep their frequency, those
                               that turn less than slow_turns times are divided by `factor`, a ramp over the pair's index
                               between (its ends rounded outwards to whole indices); cosine and sine times attention_factor */
} q4b_rotary_scaling_kind;

typedef struct q4b_rotary_scaling {
    uint32_t kind;
    uint32_t reserved;
    double factor;
    double original_length;   /* YARN */
    double fast_turns;        /* YARN, 0: 32 */
    double slow_turns;        /* YARN, 0: 1 */
    double attention_factor;  /* YARN, 0: 0.1 ln(factor) + 1 */
} q4b_rotary_scaling;

/* Radians per token of the rotary_dim / 2 pairs, base^(-2 i / rotary_dim) scaled as said (scaling null: not), and the factor on
 * cosine and sine. Host arithmetic in 64 bits; needs no runtime. */
int q4b_rotary_frequencies(uint32_t rotary_dim, double base, const q4b_rotary_scaling *scaling, double *inv_freq,
                           double *attention_factor);

typedef struct q4b_rotary q4b_rotary;

/* Keeps the frequencies (rotary_dim / 2 finite numbers, those of q4b_rotary_frequencies or the caller's own) on the device as
 * fractions of a turn in 64 bits: the angle of any int32 position is exact modulo a turn to 2^-33. rotary_dim is even, 2...256.
 * q4b_rotary_destroy waits for the device and frees them: a graph that has captured a call with the handle may not be replayed
 * behind it. */
int q4b_rotary_create(q4b_runtime *rt, const double *inv_freq, uint32_t rotary_dim, int layout, double attention_factor,
                      q4b_rotary **out);
void q4b_rotary_destroy(q4b_rotary *rotary);

/* Turns the first rotary_dim values of every head of token t by positions[t] and copies the others. `out` may be `x` (then type
 * and stride are equal too). positions_dev holds one int32 a token, negative ones turn the other way. */
int q4b_rotary_device(q4b_runtime *rt, const q4b_rotary *rotary, const void *x_dev, int x_dtype, uint64_t x_stride,
                      uint64_t tokens, uint32_t heads, uint32_t head_dim, const int32_t *positions_dev, void *out_dev,
                      int out_dtype, uint64_t out_stride, void *stream);

/* ---- paged cache of keys and values ---- */

typedef enum q4b_kv_format {
    Q4B_KV_BF16 = 0,  /* values rounded to bf16 */
    Q4B_KV_INT8 = 1,  /* code = nearest integer to x / scale, scale = max|x| / 127 over a token's head, fp32 */
    Q4B_KV_E4M3 = 2   /* code = nearest e4m3 number to x / scale, scale = max|x| / 448 */
} q4b_kv_format;

/* One layer's cache: device memory of the caller's. Value d of head h of token t of page p is at
 * p * page_stride + h * head_stride + t * token_stride + d * (size of a value), strides in bytes, multiples of 16; all three 0:
 * [pages][kv_heads][page_tokens][head_dim] without gaps. K and V have the same layout. Scales are [pages][kv_heads][page_tokens]
 * fp32 without gaps, null for bf16. All five addresses are multiples of 16 bytes. page_tokens is a multiple of 16. */
typedef struct q4b_kv_cache {
    uint32_t format;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t page_tokens;
    uint32_t pages;
    uint32_t reserved;
    void *k;
    void *v;
    float *k_scales;
    float *v_scales;
    uint64_t page_stride;
    uint64_t head_stride;
    uint64_t token_stride;
} q4b_kv_cache;

/* Which pages hold a sequence: token at position p is in page pages_dev[sequence * row_stride + p / page_tokens]. Entries that
 * no token needs are not read. row_stride 0 stands for pages_per_sequence. Sequences may share pages for reading; one call may not write
 * a place of a shared page twice (through two sequences, or two entries of one). */
typedef struct q4b_kv_table {
    const int32_t *pages_dev;
    uint32_t sequences;
    uint32_t pages_per_sequence;
    uint64_t row_stride;
} q4b_kv_table;

/* Writes `tokens` keys and values. Token t belongs to sequence sequences_dev[t] and stands at positions_dev[t] in it; a negative
 * position is a padded token: nothing is written. sequences_dev null: tokens is a multiple of the table's sequences, and they
 * have equal runs of tokens in order. Of several tokens with the same place the last one is kept. rotary, if not null, turns
 * the keys first (in 32 bits, before they are rounded). k_dev or v_dev may be null: that side is left alone. A row that holds an
 * infinity or a NaN gets a NaN for its scale, and all of it reads back as NaN (bf16 keeps such values as they are). */
int q4b_kv_write_device(q4b_runtime *rt, const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *positions_dev,
                        const int32_t *sequences_dev, uint64_t tokens, const void *k_dev, uint64_t k_stride, const void *v_dev,
                        uint64_t v_stride, int dtype, const q4b_rotary *rotary, void *stream);

/* The reverse: row t of the outputs receives what the cache holds for token t, code * scale. Rows of padded tokens (and of
 * tokens that the cache cannot hold) stay as they were. k_dev or v_dev may be null. */
int q4b_kv_read_device(q4b_runtime *rt, const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *positions_dev,
                       const int32_t *sequences_dev, uint64_t tokens, void *k_dev, uint64_t k_stride, void *v_dev,
                       uint64_t v_stride, int dtype, void *stream);

/* ---- attention ---- */

/* Attention of the last q_tokens tokens (1...16) of every sequence over its cache. Rows of q and out: sequence s, token i in row
 * s * q_tokens + i, `heads` heads each, a multiple of the cache's kv_heads; query head h reads key head
 * h / (heads / kv_heads). lengths_dev[s] counts the tokens of sequence s in the cache, the new ones among them; token i sees
 * the first lengths[s] - q_tokens + 1 + i of them:
 *     out = sum_j e^(scale q.k_j) v_j / sum_j e^(scale q.k_j).
 * A row that sees nothing (a length of 0 is a padded sequence) is zero. Products, maxima and sums are held in 32 bits, the
 * factors of each product to 16 bits or more (8-bit caches: queries to 2^-25 of the row's largest one at least, if that one
 * lies between 2^-90 and 2^100; weights times scales to 2^-26 of the largest one or to 2^-126, whichever is more). Weights
 * below 2^-125 of the row's largest one count as nothing. A number that is not finite, in a query or in keys and values,
 * reaches the rows that see it and no others. What lies behind a sequence's length in its last page is not looked at,
 * whatever it is.
 * The same call on the same data gives the same bits; another batch around a sequence may change its last bits. Tables that could
 * hold 2^32 or more 16s of tokens, over all sequences, key heads and eights of their query rows, are Q4B_DIMENSION_OVERFLOW. */
int q4b_attention_device(q4b_runtime *rt, const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *lengths_dev,
                         const void *q_dev, int q_dtype, uint64_t q_stride, uint32_t heads, uint32_t q_tokens, float scale,
                         void *out_dev, int out_dtype, uint64_t out_stride, void *stream);

#ifdef __cplusplus
}
#endif
#endif
