// C ABI of the attention step (include/openmini_attn.h): argument checks and kernel
// dispatch.  Host code only; every failure returns a status and leaves a message.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>

#include "attn_internal.hpp"

struct openmini_rope {
    attn::Rope r;
    int device = 0;
};

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return qmm::report_error(code, buf);
}

int ok() {
    qmm::set_last_error("");
    return OPENMINI_QMM_OK;
}

int launched(hipError_t e, const char* what) {
    if (e != hipSuccess) return fail(OPENMINI_QMM_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
    return ok();
}

#define TRY(expr)                                  \
    do {                                           \
        const int rc_ = (expr);                    \
        if (rc_ != OPENMINI_QMM_OK) return rc_;    \
    } while (0)

constexpr int64_t kMaxI32 = INT32_MAX;

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

int invalid(const char* what, int64_t v) {
    return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "invalid %s: %lld", what, (long long)v);
}

int check_range(const char* what, int64_t v, int64_t lo, int64_t hi) {
    if (v < lo || v > hi)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s = %lld is outside [%lld, %lld]", what, (long long)v, (long long)lo,
                    (long long)hi);
    return OPENMINI_QMM_OK;
}

int check_pointer(const char* what, const void* p, uintptr_t to) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null %s", what);
    if (!aligned(p, to)) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s is not %d-byte aligned", what, (int)to);
    return OPENMINI_QMM_OK;
}

// A stride in elements of `size` bytes: a multiple of 16 bytes, below 2^40 elements.
int check_stride(const char* what, int64_t v, int64_t least, int size) {
    if (v < least || v > ((int64_t)1 << 40) || (v * size) % 16)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s = %lld elements: at least %lld and a multiple of 16 bytes", what,
                    (long long)v, (long long)least);
    return OPENMINI_QMM_OK;
}

// Whether `count` elements of 4 bytes from p on share memory with an array of rows of `row`
// elements, `stride` from one to the next, from q on.
bool shares_memory(const void* p, int64_t count, const void* q, int64_t rows, int64_t row, int64_t stride) {
    if (!p || count <= 0) return false;
    const int64_t from = ((int64_t)(uintptr_t)p - (int64_t)(uintptr_t)q) / 4, to = from + count;  // both 4-byte aligned
    if (to <= 0 || from >= (rows - 1) * stride + row) return false;
    const int64_t r = from < 0 ? 0 : from / stride;  // the row that begins at `from` or before it
    return from < r * stride + row || (r + 1 < rows && to > (r + 1) * stride);
}

bool dense_type(int t) { return t == OPENMINI_ATTN_F32 || t == OPENMINI_ATTN_F16 || t == OPENMINI_ATTN_BF16; }
bool half_type(int t) { return t == OPENMINI_ATTN_F16 || t == OPENMINI_ATTN_BF16; }
int size_of(int t) { return t == OPENMINI_ATTN_F32 ? 4 : t == OPENMINI_ATTN_F8_E4M3 ? 1 : 2; }

int unsupported(const char* what, int t) { return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "%s: type %d is not taken", what, t); }

int check_cache(const openmini_kv_cache_t* c, attn::Cache* out) {
    if (!c) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null cache");
    if (!half_type(c->dtype) && c->dtype != OPENMINI_ATTN_F8_E4M3) return unsupported("cache", c->dtype);
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

int check_rope(const openmini_rope* rope) {
    if (!rope) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null rope handle");
    int dev = 0;
    TRY(qmm::current_device(&dev));
    if (dev != rope->device)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "rope handle lives on device %d, current device is %d", rope->device, dev);
    return OPENMINI_QMM_OK;
}

// Checks common to both rotary calls.
int check_heads(const openmini_rope* rope, int64_t tokens, int64_t heads, int64_t head_dim, const int32_t* d_positions,
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

void set_rope(attn::RopeArgs& a, const openmini_rope* rope, int64_t tokens, int heads, int kv_heads, int head_dim,
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

constexpr int kDims[] = {64, 96, 128, 192, 256};

bool decode_dim(int d) {
    for (int k : kDims)
        if (k == d) return true;
    return false;
}

size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// The workspace: the split rows, then the parts' maxima and sums, then their accumulators.
struct Workspace {
    size_t ml_at, acc_at, bytes;
};
Workspace workspace(int q_heads, int kv_heads, int head_tiles, int head_dim) {
    const size_t shares = attn::decode_shares(kv_heads, head_tiles), entries = 2 * shares * q_heads;
    Workspace w;
    w.ml_at = round_up(shares * sizeof(attn::Split), 256);
    w.acc_at = w.ml_at + round_up(entries * 8, 256);
    w.bytes = w.acc_at + entries * head_dim * 4;
    return w;
}

constexpr int64_t kMaxRows = (int64_t)1 << 20;
constexpr int64_t kMostKeys = kMaxI32 - 255;  // whole tiles of keys stay below 2^31

bool decode_sizes(int q_heads, int kv_heads, int head_dim, int* head_tiles) {
    if (kv_heads < 1 || q_heads < kv_heads || q_heads > 1024 || q_heads % kv_heads ||
        !decode_dim(head_dim))
        return false;
    const int group = q_heads / kv_heads;
    *head_tiles = (group + attn::kHeadTile - 1) / attn::kHeadTile;
    return true;
}

}  // namespace

extern "C" {

int openmini_kv_plan(const openmini_kv_plan_args_t* p, void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    TRY(check_range("requests", p->requests, 1, attn::kMaxPlanRequests));
    TRY(check_range("page_size", p->page_size, 1, (int64_t)1 << 20));
    TRY(check_range("max_pages", p->max_pages, 1, kMaxI32 / p->page_size));
    TRY(check_range("table_stride", p->table_stride, p->max_pages, (int64_t)1 << 40));
    TRY(check_range("max_tokens", p->max_tokens, 1, kMaxI32));
    TRY(check_range("n_free", p->n_free, 0, kMaxI32));
    const struct {
        const char* name;
        const void* p;
    } need[] = {{"d_cached", p->d_cached}, {"d_new", p->d_new},   {"d_tables", p->d_tables},
                {"d_starts", p->d_starts}, {"d_lens", p->d_lens}, {"d_rows", p->d_rows},
                {"d_positions", p->d_positions}, {"d_slots", p->d_slots}, {"d_row_lens", p->d_row_lens},
                {"d_counts", p->d_counts}};
    for (const auto& n : need) TRY(check_pointer(n.name, n.p, 4));
    if (p->n_free || p->d_free) TRY(check_pointer("d_free", p->d_free, 4));
    if (p->d_head) TRY(check_pointer("d_head", p->d_head, 4));
    // Every workgroup reads the inputs for itself, at its own time.
    const struct {
        const char* name;
        const void* p;
        int64_t count;
    } in[] = {{"d_cached", p->d_cached, p->requests}, {"d_new", p->d_new, p->requests}, {"d_free", p->d_free, p->n_free},
              {"d_head", p->d_head, 1}},
      out[] = {{"d_starts", p->d_starts, p->requests + 1}, {"d_lens", p->d_lens, p->requests}, {"d_rows", p->d_rows, p->max_tokens},
               {"d_positions", p->d_positions, p->max_tokens}, {"d_slots", p->d_slots, p->max_tokens},
               {"d_row_lens", p->d_row_lens, p->max_tokens}, {"d_counts", p->d_counts, 4}};
    for (const auto& i : in) {
        const char* with = shares_memory(i.p, i.count, p->d_tables, p->requests, p->max_pages, p->table_stride) ? "d_tables" : nullptr;
        for (const auto& o : out)
            if (shares_memory(i.p, i.count, o.p, 1, o.count, o.count)) with = o.name;
        if (with)
            return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "an output of the plan is one of its inputs: %s and %s share memory", i.name, with);
    }
    TRY(qmm::current_device(nullptr));
    attn::PlanArgs a;
    a.cached = p->d_cached;
    a.fresh = p->d_new;
    a.free = p->d_free;
    a.head = p->d_head;
    a.tables = p->d_tables;
    a.starts = p->d_starts;
    a.lens = p->d_lens;
    a.rows = p->d_rows;
    a.positions = p->d_positions;
    a.slots = p->d_slots;
    a.row_lens = p->d_row_lens;
    a.counts = p->d_counts;
    a.table_stride = p->table_stride;
    a.requests = (uint32_t)p->requests;
    a.n_free = (uint32_t)p->n_free;
    a.max_held = (uint32_t)(p->max_pages * p->page_size);
    a.max_tokens = (uint32_t)p->max_tokens;
    a.page = attn::FastDiv((uint32_t)p->page_size);
    return launched(attn::launch_plan(a, static_cast<hipStream_t>(stream)), "plan launch");
}

int openmini_rope_create(const double* inv_freq, const int32_t* axis, int pairs, int axes, int adjacent, float scale,
                         openmini_rope_t** out_rope) {
    if (!out_rope) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null out_rope");
    *out_rope = nullptr;
    if (!inv_freq) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null inv_freq");
    TRY(check_range("pairs", pairs, 4, attn::kMaxPairs));
    if (pairs % 4) return invalid("pairs (a multiple of 4)", pairs);
    TRY(check_range("axes", axes, 1, attn::kMaxAxes));
    if (!std::isfinite(scale)) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "scale %g is not finite", scale);
    attn::RopePair host[attn::kMaxPairs];
    for (int i = 0; i < pairs; ++i) {
        const int32_t ax = axis ? axis[i] : 0;
        if (ax < 0 || ax >= axes)
            return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "axis %d of pair %d is outside [0, %d)", ax, i, axes);
        if (!std::isfinite(inv_freq[i]))
            return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "inv_freq of pair %d is not finite", i);
        // revolutions a position, its whole part dropped, in 80-bit arithmetic
        long double turns = (long double)inv_freq[i] / 6.283185307179586476925286766559005768L;
        turns -= floorl(turns);
        const long double fixed = roundl(turns * 18446744073709551616.0L);
        host[i] = {fixed >= 18446744073709551616.0L ? 0 : (uint64_t)fixed, ax, 0};
    }
    int dev = 0;
    TRY(qmm::current_device(&dev));
    openmini_rope* h = new (std::nothrow) openmini_rope();
    if (!h) return fail(OPENMINI_QMM_ERR_MEMORY, "host allocation failed");
    void* d = nullptr;
    hipError_t e = hipMalloc(&d, sizeof(attn::RopePair) * (size_t)pairs);
    if (e != hipSuccess) {
        delete h;
        return fail(OPENMINI_QMM_ERR_MEMORY, "hipMalloc for rotary frequencies failed: %s", hipGetErrorString(e));
    }
    e = hipMemcpy(d, host, sizeof(attn::RopePair) * (size_t)pairs, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(d);
        delete h;
        return fail(OPENMINI_QMM_ERR_HIP, "copy of rotary frequencies: %s", hipGetErrorString(e));
    }
    h->device = dev;
    h->r = {static_cast<attn::RopePair*>(d), pairs, axes, adjacent != 0, scale};
    *out_rope = h;
    return ok();
}

void openmini_rope_free(openmini_rope_t* rope) {
    if (!rope) return;
    (void)hipFree(rope->r.pairs);
    delete rope;
}

int openmini_rope_apply(const openmini_rope_t* rope, const openmini_rope_args_t* p, void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    TRY(check_rope(rope));
    if (!dense_type(p->x_dtype)) return unsupported("x", p->x_dtype);
    if (!dense_type(p->y_dtype)) return unsupported("y", p->y_dtype);
    TRY(check_heads(rope, p->tokens, p->heads, p->head_dim, p->d_positions, p->position_stride));
    TRY(check_pointer("d_x", p->d_x, 16));
    TRY(check_pointer("d_y", p->d_y, 16));
    const int64_t row = (int64_t)p->heads * p->head_dim;
    TRY(check_stride("x_stride", p->x_stride, row, size_of(p->x_dtype)));
    TRY(check_stride("y_stride", p->y_stride, row, size_of(p->y_dtype)));
    if (p->d_x == p->d_y && (p->x_dtype != p->y_dtype || p->x_stride != p->y_stride))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "in place, x and y need one type and stride");
    if (p->tokens == 0) return ok();
    attn::RopeArgs a = {};
    set_rope(a, rope, p->tokens, p->heads, 0, p->head_dim, p->d_positions, p->position_stride);
    a.x = static_cast<const uint8_t*>(p->d_x);
    a.x_stride = p->x_stride * size_of(p->x_dtype);
    a.y = static_cast<uint8_t*>(p->d_y);
    a.y_stride = p->y_stride * size_of(p->y_dtype);
    a.x_dtype = p->x_dtype;
    a.y_dtype = p->y_dtype;
    a.inverse = p->inverse != 0;
    return launched(attn::launch_rope(a, p->head_dim, static_cast<hipStream_t>(stream)), "rope launch");
}

int openmini_rope_append(const openmini_rope_t* rope, const openmini_kv_cache_t* cache,
                         const openmini_rope_append_args_t* p, void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    TRY(check_rope(rope));
    attn::RopeArgs a = {};
    TRY(check_cache(cache, &a.cache));
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
    a.k_over = 1.0f / cache->k_scale;
    a.v_over = 1.0f / cache->v_scale;
    if (!std::isfinite(a.k_over) || !std::isfinite(a.v_over))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "cache scales %g, %g: below 2^-128 they have no reciprocal", cache->k_scale,
                    cache->v_scale);
    if (p->d_q_out == p->d_q || p->d_q_out == p->d_k || p->d_q_out == p->d_v)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_q_out is one of the inputs");
    if (p->tokens == 0) return ok();
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
    return launched(attn::launch_rope(a, cache->head_dim, static_cast<hipStream_t>(stream)), "rope append launch");
}

size_t openmini_attn_workspace_bytes(int q_heads, int kv_heads, int head_dim) {
    int head_tiles = 0;
    if (!decode_sizes(q_heads, kv_heads, head_dim, &head_tiles)) return 0;
    return workspace(q_heads, kv_heads, head_tiles, head_dim).bytes;
}

int openmini_attn_decode(const openmini_kv_cache_t* cache, const openmini_attn_args_t* p, void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    attn::DecodeArgs a = {};
    TRY(check_cache(cache, &a.cache));
    if (!half_type(p->q_dtype)) return unsupported("q", p->q_dtype);
    const bool f8 = cache->dtype == OPENMINI_ATTN_F8_E4M3;
    if (!f8 && cache->dtype != p->q_dtype)
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "q of type %d on a cache of type %d", p->q_dtype, cache->dtype);
    if (p->out_dtype != p->q_dtype && p->out_dtype != OPENMINI_ATTN_F32) return unsupported("out", p->out_dtype);
    if (!decode_dim(cache->head_dim))
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "head_dim = %d (64, 96, 128, 192 and 256 are taken)", cache->head_dim);
    if (cache->page_size % 8)
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "page_size = %d is not a multiple of 8", cache->page_size);
    TRY(check_range("rows", p->rows, 0, kMaxRows));
    int head_tiles = 0;
    if (!decode_sizes(p->q_heads, cache->kv_heads, cache->head_dim, &head_tiles))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "q_heads = %d for kv_heads = %d: a multiple, at most 1024", p->q_heads,
                    cache->kv_heads);
    TRY(check_pointer("d_q", p->d_q, 16));
    TRY(check_pointer("d_out", p->d_out, 16));
    TRY(check_pointer("d_lens", p->d_lens, 4));
    TRY(check_pointer("d_tables", p->d_tables, 4));
    if (p->d_rows) TRY(check_pointer("d_rows", p->d_rows, 4));
    if (p->d_lse) TRY(check_pointer("d_lse", p->d_lse, 4));
    const int64_t row = (int64_t)p->q_heads * cache->head_dim;
    const int out_size = size_of(p->out_dtype);
    TRY(check_stride("q_stride", p->q_stride, row, 2));
    TRY(check_stride("out_stride", p->out_stride, row, out_size));
    a.scale = (float)((double)p->scale * cache->k_scale * 1.44269504088896340736);
    if (!std::isfinite(a.scale))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "scale %g (times the keys' %g and log2(e)) is not finite", p->scale, cache->k_scale);
    TRY(check_range("window", p->window, 0, INT64_MAX));
    TRY(check_range("max_pages", p->max_pages, 1, kMaxI32));
    TRY(check_range("table_stride", p->table_stride, p->max_pages, (int64_t)1 << 40));
    TRY(check_range("requests", p->requests, 1, kMaxI32));
    if (p->rows == 0) return ok();
    const attn::Cache& c = a.cache;
    const int64_t held = p->max_pages * cache->page_size, max_len = held < kMostKeys ? held : kMostKeys;
    const uint32_t shares = attn::decode_shares(cache->kv_heads, head_tiles);
    // tiles of the call at most
    const int64_t tiles = p->rows * (max_len / (32 * attn::decode_subtiles(cache->head_dim, f8)) + 2);
    if (tiles > (int64_t)UINT32_MAX / 2)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%lld rows of up to %lld keys are too many for one call",
                    (long long)p->rows, (long long)max_len);
    const auto w = workspace(p->q_heads, cache->kv_heads, head_tiles, cache->head_dim);
    TRY(check_pointer("d_work", p->d_work, 256));
    if (p->work_bytes < w.bytes)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "workspace of %zu bytes, %zu are needed", p->work_bytes, w.bytes);
    TRY(qmm::current_device(nullptr));
    a.q = static_cast<const uint8_t*>(p->d_q);
    a.out = static_cast<uint8_t*>(p->d_out);
    a.lse = p->d_lse;
    a.lens = p->d_lens;
    a.rows = p->d_rows;
    a.tables = p->d_tables;
    a.q_stride = p->q_stride * 2;
    a.out_stride = p->out_stride * out_size;
    a.table_stride = p->table_stride;
    a.window = p->window && p->window < max_len ? (uint32_t)p->window : (uint32_t)max_len;
    a.n_rows = (uint32_t)p->rows;
    a.requests = (uint32_t)p->requests;
    a.max_len = (uint32_t)max_len;
    a.q_heads = p->q_heads;
    a.kv_heads = cache->kv_heads;
    a.group = p->q_heads / cache->kv_heads;
    a.head_tiles = head_tiles;
    a.out_f32 = p->out_dtype == OPENMINI_ATTN_F32;
    // the last byte that a lane's own offset reaches (heads and the eight keys of a group are
    // added to the scalar address)
    a.wide = (double)(c.n_pages - 1) * (double)c.page_stride + (double)(cache->page_size + 8) * (double)c.token_stride + 1024 >=
             4294967296.0;
    a.shares = shares;
    a.launch_shares = tiles < (int64_t)shares ? (uint32_t)tiles : shares;
    a.by_units = attn::FastDiv((uint32_t)(cache->kv_heads * head_tiles));
    a.by_head_tiles = attn::FastDiv((uint32_t)head_tiles);
    uint8_t* work = static_cast<uint8_t*>(p->d_work);
    a.split = reinterpret_cast<attn::Split*>(work);
    a.part_ml = reinterpret_cast<float2*>(work + w.ml_at);
    a.part_acc = reinterpret_cast<float*>(work + w.acc_at);
    a.by_row = p->rows <= (int64_t)shares;
    const int64_t keys = max_len < (int64_t)a.window ? max_len : (int64_t)a.window, tile = 32 * attn::decode_subtiles(cache->head_dim, f8);
    a.stream = head_tiles == 1 && p->rows <= p->requests &&
               attn::decode_streams(c, cache->kv_heads, cache->head_dim, f8, p->rows * keys);
    // a window's first tile need not begin with it
    const int64_t most = (keys + tile - 1) / tile + (keys < max_len), pairs = p->rows * cache->kv_heads * head_tiles;
    a.whole = attn::decode_whole(most, pairs);
    a.uncut = attn::decode_uncut(most, p->rows, (int64_t)cache->kv_heads * head_tiles, shares, cache->head_dim, f8);
    if (a.uncut) a.launch_shares = p->rows < (int64_t)shares ? (uint32_t)p->rows : shares;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e = p->q_dtype == OPENMINI_ATTN_BF16 ? attn::launch_decode_bf16(a, cache->head_dim, f8, s)
                                                    : attn::launch_decode_f16(a, cache->head_dim, f8, s);
    if (e == hipSuccess && !a.whole && !a.uncut && a.launch_shares > 1)
        e = attn::launch_join(a, cache->head_dim, p->out_dtype, s);
    return launched(e, "attention launch");
}

}  // extern "C"
