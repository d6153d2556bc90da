// Argument checks shared by the attention step's C ABI (attn_api.hip, attn_i8_api.hip).  Host
// code only; every failure returns a status and leaves a message.
#pragma once

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <utility>

#include "attn_internal.hpp"
#include "attn_overlap.hpp"

struct openmini_rope {
    attn::Rope r;
    int device = 0;
};

namespace attn {

inline int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return qmm::report_error(code, buf);
}

inline int ok() {
    qmm::set_last_error("");
    return OPENMINI_QMM_OK;
}

inline int launched(hipError_t e, const char* what) {
    if (e != hipSuccess) return fail(OPENMINI_QMM_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
    return ok();
}

#define TRY(expr)                                  \
    do {                                           \
        const int rc_ = (expr);                    \
        if (rc_ != OPENMINI_QMM_OK) return rc_;    \
    } while (0)

constexpr int64_t kMaxI32 = INT32_MAX;

inline bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

inline int invalid(const char* what, int64_t v) {
    return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "invalid %s: %lld", what, (long long)v);
}

inline int check_range(const char* what, int64_t v, int64_t lo, int64_t hi) {
    if (v < lo || v > hi)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s = %lld is outside [%lld, %lld]", what, (long long)v, (long long)lo,
                    (long long)hi);
    return OPENMINI_QMM_OK;
}

inline int check_pointer(const char* what, const void* p, uintptr_t to) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null %s", what);
    if (!aligned(p, to)) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s is not %d-byte aligned", what, (int)to);
    return OPENMINI_QMM_OK;
}

// A stride in elements of `size` bytes: a multiple of 16 bytes, below 2^40 elements.
inline int check_stride(const char* what, int64_t v, int64_t least, int size) {
    if (v < least || v > ((int64_t)1 << 40) || (v * size) % 16)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s = %lld elements: at least %lld and a multiple of 16 bytes", what,
                    (long long)v, (long long)least);
    return OPENMINI_QMM_OK;
}

// Whether `count` elements of 4 bytes from p on share memory with an array of rows of `row`
// elements, `stride` from one to the next, from q on.
inline bool shares_memory(const void* p, int64_t count, const void* q, int64_t rows, int64_t row, int64_t stride) {
    if (!p || count <= 0) return false;
    const int64_t from = ((int64_t)(uintptr_t)p - (int64_t)(uintptr_t)q) / 4, to = from + count;  // both 4-byte aligned
    if (to <= 0 || from >= (rows - 1) * stride + row) return false;
    const int64_t r = from < 0 ? 0 : from / stride;  // the row that begins at `from` or before it
    return from < r * stride + row || (r + 1 < rows && to > (r + 1) * stride);
}

// Bytes of a cache's keys (values), and of the scales of its keys (values).
inline Box<4> cache_bytes(const openmini_kv_cache_t* c, int size) {
    const Axis axes[] = {{1, (int64_t)c->head_dim * size}, {c->head_stride * size, c->kv_heads}, {c->token_stride * size, c->page_size},
                         {c->page_stride * size, c->n_pages}};
    return Box<4>(axes);
}
inline Box<4> scale_bytes(const openmini_kv_cache_t* c, const openmini_kv_scales_t* s) {
    const Axis axes[] = {{1, 4}, {s->head_stride * 4, c->kv_heads}, {s->block_stride * 4, c->page_size / s->block}, {s->page_stride * 4, c->n_pages}};
    return Box<4>(axes);
}
inline int64_t bytes_apart(const void* p, const void* q) { return (int64_t)((uintptr_t)p - (uintptr_t)q); }

inline bool dense_type(int t) { return t == OPENMINI_ATTN_F32 || t == OPENMINI_ATTN_F16 || t == OPENMINI_ATTN_BF16; }
inline bool half_type(int t) { return t == OPENMINI_ATTN_F16 || t == OPENMINI_ATTN_BF16; }
inline int size_of(int t) { return t == OPENMINI_ATTN_F32 ? 4 : t == OPENMINI_ATTN_F8_E4M3 || t == OPENMINI_ATTN_I8 ? 1 : 2; }

inline int unsupported(const char* what, int t) { return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "%s: type %d is not taken", what, t); }

// A cache of the types that stand by themselves, or (i8) of 8-bit integers.
inline int check_cache(const openmini_kv_cache_t* c, attn::Cache* out, bool i8 = false) {
    if (!c) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null cache");
    if (i8 ? c->dtype != OPENMINI_ATTN_I8 : !half_type(c->dtype) && c->dtype != OPENMINI_ATTN_F8_E4M3)
        return unsupported("cache", c->dtype);
    TRY(check_pointer("cache d_k", c->d_k, 16));
    TRY(check_pointer("cache d_v", c->d_v, 16));
    TRY(check_range("kv_heads", c->kv_heads, 1, 1024));
    TRY(check_range("head_dim", c->head_dim, 8, 512));
    if (c->head_dim % 8) return invalid("head_dim (a multiple of 8)", c->head_dim);
    TRY(check_range("page_size", c->page_size, 1, (int64_t)1 << 20));
    TRY(check_range("n_pages", c->n_pages, 1, kMaxI32 / c->page_size));
    const int size = size_of(c->dtype);
    TRY(check_stride("page_stride", c->page_stride, 0, size));
    TRY(check_stride("token_stride", c->token_stride, 0, size));
    TRY(check_stride("head_stride", c->head_stride, 0, size));
    if (!std::isfinite(c->k_scale) || !std::isfinite(c->v_scale) || c->k_scale <= 0 || c->v_scale <= 0)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "cache scales %g, %g: positive and finite", c->k_scale, c->v_scale);
    out->k = static_cast<uint8_t*>(c->d_k);
    out->v = static_cast<uint8_t*>(c->d_v);
    out->page_stride = c->page_stride * size;
    out->token_stride = c->token_stride * size;
    out->head_stride = c->head_stride * size;
    out->n_pages = (uint32_t)c->n_pages;
    out->slots = (uint32_t)(c->n_pages * c->page_size);
    out->page = attn::FastDiv((uint32_t)c->page_size);
    out->k_scale = c->k_scale;
    out->v_scale = c->v_scale;
    return OPENMINI_QMM_OK;
}

// A cache of 8-bit integers and its blocks' scales.
inline int check_cache_i8(const openmini_kv_cache_t* c, const openmini_kv_scales_t* s, Cache* out, Scales* to) {
    TRY(check_cache(c, out, true));
    if (c->k_scale != 1 || c->v_scale != 1)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "k_scale %g, v_scale %g of a cache of 8-bit integers: 1", c->k_scale, c->v_scale);
    if (!s) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null scales");
    TRY(check_pointer("scales d_k", s->d_k, 4));
    TRY(check_pointer("scales d_v", s->d_v, 4));
    if (s->block != 8 && s->block != 16 && s->block != 32) return invalid("block (8, 16 or 32)", s->block);
    if (c->page_size % s->block)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "page_size = %d is not a multiple of the block of %d", c->page_size, s->block);
    // from the smallest stride on, each passes over what the ones before it reach
    struct {
        int64_t stride, count;
    } d[] = {{s->page_stride, c->n_pages}, {s->block_stride, c->page_size / s->block}, {s->head_stride, c->kv_heads}};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j)
            if (d[j].stride > d[j + 1].stride) std::swap(d[j], d[j + 1]);
    double reach = 1;  // exact where a stride can be as much; their sum may pass 63 bits
    for (const auto& x : d) {
        if (x.stride < 0 || x.stride > ((int64_t)1 << 40) || (x.count > 1 && (double)x.stride < reach))
            return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "scales' strides %lld, %lld, %lld: two scales share an element",
                        (long long)s->page_stride, (long long)s->block_stride, (long long)s->head_stride);
        reach += (double)x.stride * (double)(x.count - 1);
    }
    to->k = s->d_k;
    to->v = s->d_v;
    to->page_stride = s->page_stride;
    to->block_stride = s->block_stride;
    to->head_stride = s->head_stride;
    to->shift = s->block == 8 ? 3 : s->block == 16 ? 4 : 5;
    return OPENMINI_QMM_OK;
}

// Any cache; `scales` are for 8-bit integers alone.
inline int check_any_cache(const openmini_kv_cache_t* c, const openmini_kv_scales_t* s, Cache* out, Scales* to) {
    if (c && c->dtype == OPENMINI_ATTN_I8) return check_cache_i8(c, s, out, to);
    TRY(check_cache(c, out));
    if (s) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "scales for a cache of type %d", c->dtype);
    return OPENMINI_QMM_OK;
}

inline int check_rope(const openmini_rope* rope) {
    if (!rope) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null rope handle");
    int dev = 0;
    TRY(qmm::current_device(&dev));
    if (dev != rope->device)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "rope handle lives on device %d, current device is %d", rope->device, dev);
    return OPENMINI_QMM_OK;
}

// Checks common to both rotary calls.
inline int check_heads(const openmini_rope* rope, int64_t tokens, int64_t heads, int64_t head_dim, const int32_t* d_positions,
                int64_t position_stride) {
    TRY(check_range("tokens", tokens, 0, kMaxI32));
    TRY(check_range("heads", heads, 1, 4096));
    TRY(check_range("head_dim", head_dim, 8, 512));
    if (head_dim % 8) return invalid("head_dim (a multiple of 8)", head_dim);
    if (2 * rope->r.n_pairs > head_dim)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%d rotary pairs do not fit head_dim = %lld", rope->r.n_pairs,
                    (long long)head_dim);
    TRY(check_pointer("d_positions", d_positions, 4));
    if (rope->r.axes > 1 && position_stride < tokens)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "position_stride = %lld below the %lld tokens", (long long)position_stride,
                    (long long)tokens);
    return OPENMINI_QMM_OK;
}

inline void set_rope(attn::RopeArgs& a, const openmini_rope* rope, int64_t tokens, int heads, int kv_heads, int head_dim,
              const int32_t* d_positions, int64_t position_stride) {
    a.positions = d_positions;
    a.position_stride = position_stride;
    a.pairs = rope->r.pairs;
    a.scale = rope->r.scale;
    a.n_pairs = rope->r.n_pairs;
    a.adjacent = rope->r.adjacent;
    a.tokens = (int32_t)tokens;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.per_head = attn::FastDiv((uint32_t)head_dim / 8);
    a.per_token = attn::FastDiv((uint32_t)((heads + 2 * kv_heads) * (head_dim / 8)));
    a.by_pairs = attn::FastDiv((uint32_t)rope->r.n_pairs);
}

// Checks common to both appending calls, and what their kernels share of the arguments.
inline int check_append(const openmini_rope* rope, const openmini_kv_cache_t* cache, const openmini_rope_append_args_t* p) {
    if (!dense_type(p->in_dtype)) return unsupported("q, k, v", p->in_dtype);
    if (!half_type(p->q_out_dtype)) return unsupported("q_out", p->q_out_dtype);
    TRY(check_heads(rope, p->tokens, p->q_heads, cache->head_dim, p->d_positions, p->position_stride));
    TRY(check_pointer("d_q", p->d_q, 16));
    TRY(check_pointer("d_k", p->d_k, 16));
    TRY(check_pointer("d_v", p->d_v, 16));
    TRY(check_pointer("d_q_out", p->d_q_out, 16));
    TRY(check_pointer("d_slots", p->d_slots, 4));
    const int in = size_of(p->in_dtype);
    const int64_t q_row = (int64_t)p->q_heads * cache->head_dim, kv_row = (int64_t)cache->kv_heads * cache->head_dim;
    TRY(check_stride("q_stride", p->q_stride, q_row, in));
    TRY(check_stride("k_stride", p->k_stride, kv_row, in));
    TRY(check_stride("v_stride", p->v_stride, kv_row, in));
    TRY(check_stride("q_out_stride", p->q_out_stride, q_row, 2));
    if (p->d_q_out == p->d_q || p->d_q_out == p->d_k || p->d_q_out == p->d_v)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_q_out is one of the inputs");
    return OPENMINI_QMM_OK;
}

inline void set_append(attn::RopeArgs& a, const openmini_rope* rope, const openmini_kv_cache_t* cache,
                       const openmini_rope_append_args_t* p) {
    const int in = size_of(p->in_dtype);
    set_rope(a, rope, p->tokens, p->q_heads, cache->kv_heads, cache->head_dim, p->d_positions, p->position_stride);
    a.x = static_cast<const uint8_t*>(p->d_q);
    a.k = static_cast<const uint8_t*>(p->d_k);
    a.v = static_cast<const uint8_t*>(p->d_v);
    a.x_stride = p->q_stride * in;
    a.k_stride = p->k_stride * in;
    a.v_stride = p->v_stride * in;
    a.y = static_cast<uint8_t*>(p->d_q_out);
    a.y_stride = p->q_out_stride * 2;
    a.x_dtype = p->in_dtype;
    a.y_dtype = p->q_out_dtype;
    a.cache_dtype = cache->dtype;
    a.slots = p->d_slots;
}

constexpr int kDims[] = {64, 96, 128, 192, 256};

inline bool decode_dim(int d) {
    for (int k : kDims)
        if (k == d) return true;
    return false;
}

inline size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

constexpr int64_t kMaxRows = (int64_t)1 << 20;
constexpr int64_t kMostKeys = kMaxI32 - 255;  // whole tiles of keys stay below 2^31

}  // namespace attn
