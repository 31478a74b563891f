// C entry points of the attention operators (include/q4b_attention.h): checks of arguments, frequencies of rotary positions, and
// launches of the kernels in q4_kv_cache.cu and q4_attention.cu.
#include "../../include/q4b_attention.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <new>

#include "q4_attention.h"

struct q4b_rotary {
    int device = 0;
    uint32_t pairs = 0, interleaved = 0;
    float factor = 1.f;
    uint64_t *step = nullptr;  // device
};

namespace {

constexpr uint64_t kMaxTokens = 0x7fffffffull;  // blocks of a launch

int fail(int status, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return q4::set_error(status, buf);
}

int launched(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return Q4B_OK;
    cudaGetLastError();  // (or the next call's launch would report it again)
    return fail(Q4B_CUDA_ERROR, "CUDA call failed in %s: %s", what, cudaGetErrorString(e));
}

// A range of device memory that a call reads or writes: [begin, end).
struct Span {
    uintptr_t begin = 0, end = 0;
    Span() = default;
    Span(const void *p, uint64_t bytes) : begin((uintptr_t)p), end((uintptr_t)p + bytes) {}
    bool meets(const Span &o) const { return begin < o.end && o.begin < end; }
};

// a * b; false when that is above 2^62
bool product(uint64_t a, uint64_t b, uint64_t *out) {
    if (b != 0 && a > (1ull << 62) / b) return false;
    *out = a * b;
    return true;
}

int check_type(int dtype) {
    if (dtype != Q4B_F32 && dtype != Q4B_BF16) return fail(Q4B_INVALID_ARGUMENT, "unknown activation dtype %d", dtype);
    return Q4B_OK;
}

int check_head_dim(uint32_t head_dim) {
    if (head_dim == 0) return fail(Q4B_EMPTY_DIMENSION, "head_dim must be greater than zero");
    if (head_dim % 16 != 0 || head_dim > q4::kMaxHeadDim) return fail(Q4B_UNSUPPORTED, "head_dim %u is not a multiple of 16 up to %u", head_dim, q4::kMaxHeadDim);
    return Q4B_OK;
}

// rows of tokens: type, alignment, stride; *span is what they cover
int check_rows(const char *name, const void *ptr, int dtype, uint64_t tokens, uint32_t heads, uint32_t head_dim, uint64_t stride, Span *span) {
    if (int st = check_type(dtype)) return st;
    if (!ptr) return fail(Q4B_INVALID_ARGUMENT, "%s pointer is null", name);
    const uint64_t size = dtype == Q4B_F32 ? 4 : 2, width = (uint64_t)heads * head_dim;
    uint64_t bytes;
    if (!product(stride, size, &bytes) || !product(bytes, tokens, &bytes) || (uintptr_t)ptr > (1ull << 62)) return fail(Q4B_DIMENSION_OVERFLOW, "%s exceeds runtime limits", name);
    if (((uintptr_t)ptr & 15u) || (stride * size) % 16 != 0) return fail(Q4B_INVALID_ARGUMENT, "%s must start at, and step by, multiples of 16 bytes", name);
    if (stride < width && tokens > 1) return fail(Q4B_WRONG_LENGTH, "%s stride has %llu elements, expected at least %llu", name, (unsigned long long)stride, (unsigned long long)width);
    *span = Span(ptr, ((tokens - 1) * stride + width) * size);
    return Q4B_OK;
}

uint32_t value_bytes(uint32_t format) { return format == Q4B_KV_BF16 ? 2u : 1u; }

struct CacheSpans {
    Span k, v, k_scales, v_scales, table;
    bool meets(const Span &s) const { return k.meets(s) || v.meets(s) || k_scales.meets(s) || v_scales.meets(s); }
};

// Checks cache and page table and describes them for the kernels.
int check_cache(const q4b_kv_cache *c, const q4b_kv_table *t, bool need_k, bool need_v, q4::KvView *view, CacheSpans *spans) {
    if (!c || !t) return fail(Q4B_INVALID_ARGUMENT, "cache or page table pointer is null");
    if (c->format > Q4B_KV_E4M3) return fail(Q4B_INVALID_ARGUMENT, "unknown cache format %u", c->format);
    if (c->kv_heads == 0 || c->page_tokens == 0 || c->pages == 0 || t->sequences == 0 || t->pages_per_sequence == 0)
        return fail(Q4B_EMPTY_DIMENSION, "cache dimensions must be greater than zero");
    if (int st = check_head_dim(c->head_dim)) return st;
    if (c->page_tokens % 16 != 0) return fail(Q4B_UNSUPPORTED, "page_tokens %u is not a multiple of 16", c->page_tokens);
    if (c->kv_heads > 65535u || c->page_tokens > (1u << 20) || c->pages > 0x7fffffffu || t->sequences > 0x7fffffffu)
        return fail(Q4B_DIMENSION_OVERFLOW, "cache dimensions exceed runtime limits");
    if ((uint64_t)t->pages_per_sequence * c->page_tokens > 0x7fffffffull) return fail(Q4B_DIMENSION_OVERFLOW, "positions of the page table exceed 2^31 - 1");
    const bool scaled = c->format != Q4B_KV_BF16;
    if ((need_k && !c->k) || (need_v && !c->v) || !t->pages_dev) return fail(Q4B_INVALID_ARGUMENT, "cache pointer is null");
    if (scaled && ((need_k && !c->k_scales) || (need_v && !c->v_scales))) return fail(Q4B_INVALID_ARGUMENT, "scales of a quantised cache are null");
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 15u) return fail(Q4B_INVALID_ARGUMENT, "cache addresses must be 16-byte aligned");
    if ((uintptr_t)t->pages_dev & 3u) return fail(Q4B_INVALID_ARGUMENT, "page table must be 4-byte aligned");
    const uint64_t row = (uint64_t)c->head_dim * value_bytes(c->format);
    uint64_t stride[3] = {c->token_stride, c->head_stride, c->page_stride};
    const uint64_t count[3] = {c->page_tokens, c->kv_heads, c->pages};
    if (!stride[0] && !stride[1] && !stride[2]) {
        stride[0] = row;
        stride[1] = row * count[0];
        if (!product(stride[1], count[1], &stride[2])) return fail(Q4B_DIMENSION_OVERFLOW, "cache exceeds runtime limits");
    }
    // tokens, heads and pages lie inside one another in some order, so that no two of them share memory
    uint32_t order[3] = {0, 1, 2};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2 - i; ++j)
            if (stride[order[j]] > stride[order[j + 1]]) {
                const uint32_t o = order[j];
                order[j] = order[j + 1];
                order[j + 1] = o;
            }
    uint64_t extent = row;
    for (uint32_t o : order) {
        if (stride[o] % 16 != 0) return fail(Q4B_INVALID_ARGUMENT, "cache strides must be multiples of 16 bytes");
        if (stride[o] >= (1ull << 40)) return fail(Q4B_DIMENSION_OVERFLOW, "cache strides exceed runtime limits");
        if (count[o] == 1) continue;
        if (stride[o] < extent) return fail(Q4B_INVALID_ARGUMENT, "cache strides let rows of the cache share memory");
        uint64_t more;
        if (!product(count[o] - 1, stride[o], &more) || more > (1ull << 61)) return fail(Q4B_DIMENSION_OVERFLOW, "cache exceeds runtime limits");
        extent += more;
    }
    const uint64_t entries = t->row_stride ? t->row_stride : t->pages_per_sequence;
    if (entries < t->pages_per_sequence && t->sequences > 1)
        return fail(Q4B_WRONG_LENGTH, "page table stride has %llu elements, expected at least %u", (unsigned long long)entries, t->pages_per_sequence);
    uint64_t table_bytes;
    if (!product(entries, t->sequences, &table_bytes) || !product(table_bytes, 4, &table_bytes)) return fail(Q4B_DIMENSION_OVERFLOW, "page table exceeds runtime limits");
    const uint64_t scale_bytes = (uint64_t)c->pages * c->kv_heads * c->page_tokens * 4;
    if (need_k) spans->k = Span(c->k, extent);
    if (need_v) spans->v = Span(c->v, extent);
    if (need_k && scaled) spans->k_scales = Span(c->k_scales, scale_bytes);
    if (need_v && scaled) spans->v_scales = Span(c->v_scales, scale_bytes);
    spans->table = Span(t->pages_dev, ((t->sequences - 1) * entries + t->pages_per_sequence) * 4);
    memset(view, 0, sizeof *view);
    view->k = (uint8_t *)c->k;
    view->v = (uint8_t *)c->v;
    view->k_scales = c->k_scales;
    view->v_scales = c->v_scales;
    view->token_stride = stride[0];
    view->head_stride = stride[1];
    view->page_stride = stride[2];
    view->format = c->format;
    view->kv_heads = c->kv_heads;
    view->head_dim = c->head_dim;
    view->page_tokens = c->page_tokens;
    view->pages = c->pages;
    view->table = t->pages_dev;
    view->sequences = t->sequences;
    view->per_sequence = t->pages_per_sequence;
    view->row_stride = entries;
    return Q4B_OK;
}

// Whether a row of the keys and one of the values share memory. Tokens, heads and pages lie inside one another, so that along each of them,
// from the widest on, only the two steps nearest to the distance come near enough.
bool rows_meet(const q4::KvView &kv, int64_t apart) {
    struct Axis {
        int64_t stride, count;
    } axis[3] = {{(int64_t)kv.token_stride, kv.page_tokens}, {(int64_t)kv.head_stride, kv.kv_heads}, {(int64_t)kv.page_stride, kv.pages}};
    std::sort(axis, axis + 3, [](const Axis &a, const Axis &b) { return a.stride > b.stride; });
    const int64_t row = (int64_t)kv.head_dim * value_bytes(kv.format);
    for (int pick = 0; pick < 8; ++pick) {
        int64_t left = apart;
        bool there = true;
        for (int i = 0; i < 3; ++i) {
            if (axis[i].count == 1) continue;
            int64_t step = left / axis[i].stride - (left % axis[i].stride < 0) + (pick >> i & 1);
            there = there && step < axis[i].count && -step < axis[i].count;
            left -= step * axis[i].stride;
        }
        if (there && left < row && -left < row) return true;
    }
    return false;
}

int check_index(const char *name, const int32_t *ptr, uint64_t count, Span *span) {
    if (!ptr) return fail(Q4B_INVALID_ARGUMENT, "%s pointer is null", name);
    if ((uintptr_t)ptr & 3u) return fail(Q4B_INVALID_ARGUMENT, "%s must be 4-byte aligned", name);
    *span = Span(ptr, count * 4);
    return Q4B_OK;
}

int check_rotary(const q4b_rotary *rotary, uint32_t head_dim, int device, q4::RotaryView *view) {
    if (2 * rotary->pairs > head_dim) return fail(Q4B_WRONG_LENGTH, "rotary pairs have %u elements, head_dim is %u", 2 * rotary->pairs, head_dim);
    if (rotary->device != device) return fail(Q4B_INVALID_ARGUMENT, "rotary frequencies are on device %d, the runtime is on %d", rotary->device, device);
    view->step = rotary->step;
    view->pairs = rotary->pairs;
    view->interleaved = rotary->interleaved;
    view->factor = rotary->factor;
    return Q4B_OK;
}

int check_rt(q4b_runtime *rt) {
    if (!rt) return fail(Q4B_INVALID_ARGUMENT, "runtime handle is null");
    return Q4B_OK;
}

int check_tokens(uint64_t tokens) {
    if (tokens == 0) return fail(Q4B_EMPTY_DIMENSION, "tokens must be greater than zero");
    if (tokens > kMaxTokens) return fail(Q4B_DIMENSION_OVERFLOW, "tokens exceed runtime limits");
    return Q4B_OK;
}

// what write and read share; k and v are the activations, either may be null
int check_kv_tokens(const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *positions, const int32_t *sequences,
                    uint64_t tokens, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride, int dtype, q4::KvTokensParams *p,
                    CacheSpans *spans, Span rows[2], Span index[2]) {
    if (int st = check_tokens(tokens)) return st;
    if (!k && !v) return fail(Q4B_INVALID_ARGUMENT, "keys and values are both null");
    memset(p, 0, sizeof *p);
    if (int st = check_cache(cache, table, k != nullptr, v != nullptr, &p->kv, spans)) return st;
    if (k)
        if (int st = check_rows("keys", k, dtype, tokens, cache->kv_heads, cache->head_dim, k_stride, &rows[0])) return st;
    if (v)
        if (int st = check_rows("values", v, dtype, tokens, cache->kv_heads, cache->head_dim, v_stride, &rows[1])) return st;
    if (int st = check_index("positions", positions, tokens, &index[0])) return st;
    if (sequences) {
        if (int st = check_index("sequences", sequences, tokens, &index[1])) return st;
    } else if (tokens % table->sequences != 0) {
        return fail(Q4B_WRONG_LENGTH, "tokens has %llu elements, expected a multiple of %u sequences", (unsigned long long)tokens, table->sequences);
    }
    p->positions = positions;
    p->sequences = sequences;
    p->tokens = tokens;
    p->run = (uint32_t)(tokens / table->sequences);
    p->k_stride = k_stride;
    p->v_stride = v_stride;
    p->is_f32 = dtype == Q4B_F32;
    return Q4B_OK;
}

}  // namespace

// ------------------------------------------------------------------------------------------
// rotary positions
// ------------------------------------------------------------------------------------------

extern "C" int q4b_rotary_frequencies(uint32_t rotary_dim, double base, const q4b_rotary_scaling *scaling, double *inv_freq, double *attention_factor) {
    if (!inv_freq || !attention_factor) return fail(Q4B_INVALID_ARGUMENT, "frequency pointer is null");
    if (rotary_dim == 0) return fail(Q4B_EMPTY_DIMENSION, "rotary_dim must be greater than zero");
    if (rotary_dim % 2 != 0 || rotary_dim > q4::kMaxHeadDim) return fail(Q4B_UNSUPPORTED, "rotary_dim %u is not an even number up to %u", rotary_dim, q4::kMaxHeadDim);
    if (!std::isfinite(base) || base <= 1.0) return fail(Q4B_INVALID_ARGUMENT, "rotary base must be a number above 1");
    const uint32_t kind = scaling ? scaling->kind : Q4B_ROTARY_UNSCALED;
    if (kind > Q4B_ROTARY_YARN) return fail(Q4B_INVALID_ARGUMENT, "unknown rotary scaling %u", kind);
    const double factor = kind ? scaling->factor : 1.0, dim = rotary_dim;
    if (!std::isfinite(factor) || factor <= 0.0) return fail(Q4B_INVALID_ARGUMENT, "rotary scaling factor must be a number above 0");
    const double pi = 3.14159265358979323846;
    double low = 0.0, high = 0.0, amplitude = 1.0;
    if (kind == Q4B_ROTARY_NTK && rotary_dim > 2) base *= std::pow(factor, dim / (dim - 2.0));
    if (kind == Q4B_ROTARY_YARN) {
        const double fast = scaling->fast_turns != 0.0 ? scaling->fast_turns : 32.0, slow = scaling->slow_turns != 0.0 ? scaling->slow_turns : 1.0;
        if (!std::isfinite(scaling->original_length) || scaling->original_length <= 0.0 || !std::isfinite(fast) || !std::isfinite(slow) || !(fast > slow) || slow <= 0.0 ||
            !std::isfinite(scaling->attention_factor) || scaling->attention_factor < 0.0)
            return fail(Q4B_INVALID_ARGUMENT, "rotary scaling needs an original length, fast_turns above slow_turns above 0, and an attention factor of 0 or more");
        // index of the pair that turns so many times in the original length
        auto edge = [&](double turns) { return dim * std::log(scaling->original_length / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
        low = std::fmax(std::floor(edge(fast)), 0.0);
        high = std::fmin(std::ceil(edge(slow)), dim - 1.0);
        amplitude = scaling->attention_factor != 0.0 ? scaling->attention_factor : (factor > 1.0 ? 0.1 * std::log(factor) + 1.0 : 1.0);
    }
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / dim);
        if (kind == Q4B_ROTARY_LINEAR) f /= factor;
        if (kind == Q4B_ROTARY_YARN) {
            const double ramp = std::fmin(std::fmax((i - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        inv_freq[i] = f;
    }
    *attention_factor = amplitude;
    return Q4B_OK;
}

extern "C" int q4b_rotary_create(q4b_runtime *rt, const double *inv_freq, uint32_t rotary_dim, int layout, double attention_factor, q4b_rotary **out) {
    if (!out) return fail(Q4B_INVALID_ARGUMENT, "output handle pointer is null");
    *out = nullptr;
    if (!inv_freq) return fail(Q4B_INVALID_ARGUMENT, "frequency pointer is null");
    if (rotary_dim == 0) return fail(Q4B_EMPTY_DIMENSION, "rotary_dim must be greater than zero");
    if (rotary_dim % 2 != 0 || rotary_dim > q4::kMaxHeadDim) return fail(Q4B_UNSUPPORTED, "rotary_dim %u is not an even number up to %u", rotary_dim, q4::kMaxHeadDim);
    if (layout != Q4B_ROTARY_HALF && layout != Q4B_ROTARY_INTERLEAVED) return fail(Q4B_INVALID_ARGUMENT, "unknown rotary layout %d", layout);
    if (!std::isfinite(attention_factor) || !std::isfinite((float)attention_factor)) return fail(Q4B_INVALID_ARGUMENT, "attention factor is not a number of 32 bits");
    uint64_t step[q4::kMaxHeadDim / 2];
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        if (!std::isfinite(inv_freq[i])) return fail(Q4B_INVALID_ARGUMENT, "frequency %u is not finite", i);
        // turns per token, as a fraction of 2^64 (a whole turn more or less does not matter to a whole number of tokens)
        long double turns = (long double)inv_freq[i] / 6.283185307179586476925286766559L;
        turns -= floorl(turns);
        const long double scaled = floorl(turns * 18446744073709551616.0L + 0.5L);
        step[i] = scaled >= 18446744073709551616.0L ? 0ull : (uint64_t)scaled;
    }
    if (int st = check_rt(rt)) return st;
    const q4::RuntimeView v = q4::runtime_view(rt);
    std::lock_guard<std::recursive_mutex> lock(*v.mu);
    q4::DeviceGuard guard(v.device);
    q4b_rotary *r = new (std::nothrow) q4b_rotary();
    if (!r) return fail(Q4B_CUDA_ERROR, "out of host memory");
    r->device = v.device;
    r->pairs = rotary_dim / 2;
    r->interleaved = layout == Q4B_ROTARY_INTERLEAVED;
    r->factor = (float)attention_factor;
    cudaError_t e = cudaMalloc((void **)&r->step, r->pairs * sizeof(uint64_t));
    // (a copy from pageable memory of this size has been read when the call returns; the legacy stream's end is waited for below)
    if (e == cudaSuccess) e = cudaMemcpy(r->step, step, r->pairs * sizeof(uint64_t), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
    if (e != cudaSuccess) {
        if (r->step) cudaFree(r->step);
        delete r;
        return launched(e, "rotary frequencies");
    }
    *out = r;
    return Q4B_OK;
}

extern "C" void q4b_rotary_destroy(q4b_rotary *rotary) {
    if (!rotary) return;
    q4::DeviceGuard guard(rotary->device);
    cudaDeviceSynchronize();
    cudaFree(rotary->step);
    delete rotary;
}

extern "C" int q4b_rotary_device(q4b_runtime *rt, const q4b_rotary *rotary, const void *x_dev, int x_dtype, uint64_t x_stride, uint64_t tokens, uint32_t heads,
                                 uint32_t head_dim, const int32_t *positions_dev, void *out_dev, int out_dtype, uint64_t out_stride, void *stream) {
    if (int st = check_tokens(tokens)) return st;
    if (heads == 0) return fail(Q4B_EMPTY_DIMENSION, "heads must be greater than zero");
    if (heads > 65535u) return fail(Q4B_DIMENSION_OVERFLOW, "heads exceed runtime limits");
    if (int st = check_head_dim(head_dim)) return st;
    Span x, out, index;
    if (int st = check_rows("input", x_dev, x_dtype, tokens, heads, head_dim, x_stride, &x)) return st;
    if (int st = check_rows("output", out_dev, out_dtype, tokens, heads, head_dim, out_stride, &out)) return st;
    if (int st = check_index("positions", positions_dev, tokens, &index)) return st;
    const bool in_place = out_dev == x_dev && x_dtype == out_dtype && (x_stride == out_stride || tokens == 1);
    if ((out.meets(x) && !in_place) || out.meets(index)) return fail(Q4B_INVALID_ARGUMENT, "output shares memory with an input");
    if (!rotary) return fail(Q4B_INVALID_ARGUMENT, "rotary handle is null");
    if (int st = check_rt(rt)) return st;
    const q4::RuntimeView v = q4::runtime_view(rt);
    q4::RotaryParams p;
    memset(&p, 0, sizeof p);
    if (int st = check_rotary(rotary, head_dim, v.device, &p.rotary)) return st;
    p.x = x_dev;
    p.out = out_dev;
    p.positions = positions_dev;
    p.x_stride = x_stride;
    p.out_stride = out_stride;
    p.tokens = tokens;
    p.heads = heads;
    p.head_dim = head_dim;
    p.x_is_f32 = x_dtype == Q4B_F32;
    p.out_is_f32 = out_dtype == Q4B_F32;
    std::lock_guard<std::recursive_mutex> lock(*v.mu);
    q4::DeviceGuard guard(v.device);
    if (int st = launched(q4k_rotary(&p, (uint32_t)v.sm_count, (cudaStream_t)stream), "rotary launch")) return st;
    ++*v.launches;
    return Q4B_OK;
}

// ------------------------------------------------------------------------------------------
// paged cache
// ------------------------------------------------------------------------------------------

extern "C" int q4b_kv_write_device(q4b_runtime *rt, const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *positions_dev, const int32_t *sequences_dev,
                                   uint64_t tokens, const void *k_dev, uint64_t k_stride, const void *v_dev, uint64_t v_stride, int dtype, const q4b_rotary *rotary,
                                   void *stream) {
    q4::KvTokensParams p;
    CacheSpans spans;
    Span rows[2], index[2];
    if (int st = check_kv_tokens(cache, table, positions_dev, sequences_dev, tokens, k_dev, k_stride, v_dev, v_stride, dtype, &p, &spans, rows, index)) return st;
    if (k_dev && v_dev && (rows_meet(p.kv, (int64_t)((uintptr_t)cache->v - (uintptr_t)cache->k)) || spans.k_scales.meets(spans.v_scales)))
        return fail(Q4B_INVALID_ARGUMENT, "keys and values of the cache share memory");
    if (spans.meets(rows[0]) || spans.meets(rows[1]) || spans.meets(index[0]) || spans.meets(index[1]) || spans.meets(spans.table))
        return fail(Q4B_INVALID_ARGUMENT, "cache shares memory with an input");
    if (int st = check_rt(rt)) return st;
    const q4::RuntimeView v = q4::runtime_view(rt);
    if (rotary)
        if (int st = check_rotary(rotary, cache->head_dim, v.device, &p.rotary)) return st;
    p.k_in = k_dev;
    p.v_in = v_dev;
    p.kv.input_error = v.input_error;
    std::lock_guard<std::recursive_mutex> lock(*v.mu);
    q4::DeviceGuard guard(v.device);
    if (int st = launched(q4k_kv_write(&p, (uint32_t)v.sm_count, (cudaStream_t)stream), "cache write launch")) return st;
    ++*v.launches;
    return Q4B_OK;
}

extern "C" int q4b_kv_read_device(q4b_runtime *rt, const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *positions_dev, const int32_t *sequences_dev,
                                  uint64_t tokens, void *k_dev, uint64_t k_stride, void *v_dev, uint64_t v_stride, int dtype, void *stream) {
    q4::KvTokensParams p;
    CacheSpans spans;
    Span rows[2], index[2];
    if (int st = check_kv_tokens(cache, table, positions_dev, sequences_dev, tokens, k_dev, k_stride, v_dev, v_stride, dtype, &p, &spans, rows, index)) return st;
    if (rows[0].meets(rows[1])) {
        // keys and values of a token may stand beside each other in rows of one stride
        const uint64_t size = dtype == Q4B_F32 ? 4 : 2, width = (uint64_t)cache->kv_heads * cache->head_dim * size, step = k_stride * size;
        const uint64_t apart = rows[0].begin < rows[1].begin ? rows[1].begin - rows[0].begin : rows[0].begin - rows[1].begin;
        if (tokens == 1 || k_stride != v_stride || apart % step < width || step - apart % step < width) return fail(Q4B_INVALID_ARGUMENT, "outputs share memory");
    }
    for (const Span &out : {rows[0], rows[1]})
        if (spans.meets(out) || index[0].meets(out) || index[1].meets(out) || spans.table.meets(out)) return fail(Q4B_INVALID_ARGUMENT, "output shares memory with an input");
    if (int st = check_rt(rt)) return st;
    const q4::RuntimeView v = q4::runtime_view(rt);
    p.k_out = k_dev;
    p.v_out = v_dev;
    p.kv.input_error = v.input_error;
    std::lock_guard<std::recursive_mutex> lock(*v.mu);
    q4::DeviceGuard guard(v.device);
    if (int st = launched(q4k_kv_read(&p, (uint32_t)v.sm_count, (cudaStream_t)stream), "cache read launch")) return st;
    ++*v.launches;
    return Q4B_OK;
}

// ------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------

extern "C" int q4b_attention_device(q4b_runtime *rt, const q4b_kv_cache *cache, const q4b_kv_table *table, const int32_t *lengths_dev, const void *q_dev, int q_dtype,
                                    uint64_t q_stride, uint32_t heads, uint32_t q_tokens, float scale, void *out_dev, int out_dtype, uint64_t out_stride, void *stream) {
    q4::AttentionParams p;
    memset(&p, 0, sizeof p);
    CacheSpans spans;
    if (int st = check_cache(cache, table, true, true, &p.kv, &spans)) return st;
    if (heads == 0 || q_tokens == 0) return fail(Q4B_EMPTY_DIMENSION, "heads and q_tokens must be greater than zero");
    if (heads > 65535u) return fail(Q4B_DIMENSION_OVERFLOW, "heads exceed runtime limits");
    if (heads % cache->kv_heads != 0) return fail(Q4B_WRONG_LENGTH, "heads has %u elements, expected a multiple of %u", heads, cache->kv_heads);
    if (q_tokens > 16u) return fail(Q4B_UNSUPPORTED, "q_tokens %u is above 16", q_tokens);
    if (!std::isfinite(scale)) return fail(Q4B_INVALID_ARGUMENT, "scale is not finite");
    const uint64_t rows = (uint64_t)table->sequences * q_tokens;
    if (rows > kMaxTokens) return fail(Q4B_DIMENSION_OVERFLOW, "tokens exceed runtime limits");
    // 16-token tiles of all key heads and groups of eight query rows, at the longest lengths: numbered in 32 bits
    const uint64_t tiles = (uint64_t)table->pages_per_sequence * (cache->page_tokens / 16), chunks = ((uint64_t)(heads / cache->kv_heads) * q_tokens + 7) / 8;
    uint64_t work;
    if (!product(tiles, table->sequences, &work) || !product(work, cache->kv_heads * chunks, &work) || work > 0xffffffffull)
        return fail(Q4B_DIMENSION_OVERFLOW, "sequences, heads and page table have room for 2^32 or more tiles of 16 tokens");
    Span q, out, lengths;
    if (int st = check_rows("queries", q_dev, q_dtype, rows, heads, cache->head_dim, q_stride, &q)) return st;
    if (int st = check_rows("output", out_dev, out_dtype, rows, heads, cache->head_dim, out_stride, &out)) return st;
    if (int st = check_index("lengths", lengths_dev, table->sequences, &lengths)) return st;
    if (out.meets(q) || out.meets(lengths) || out.meets(spans.table) || spans.meets(out)) return fail(Q4B_INVALID_ARGUMENT, "output shares memory with an input");
    if (int st = check_rt(rt)) return st;
    const q4::RuntimeView v = q4::runtime_view(rt);
    p.lengths = lengths_dev;
    p.q = q_dev;
    p.out = out_dev;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.heads = heads;
    p.q_tokens = q_tokens;
    p.q_is_f32 = q_dtype == Q4B_F32;
    p.out_is_f32 = out_dtype == Q4B_F32;
    p.scale = scale;
    p.parts = v.attention_parts;
    p.counters = v.attention_counters;
    p.error_flag = v.error_flag;
    p.kv.input_error = v.input_error;
    std::lock_guard<std::recursive_mutex> lock(*v.mu);
    q4::DeviceGuard guard(v.device);
    if (int st = launched(q4k_attention(&p, (uint32_t)v.sm_count, (cudaStream_t)stream), "attention launch")) return st;
    ++*v.launches;
    return Q4B_OK;
}
