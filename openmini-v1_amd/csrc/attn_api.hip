// C ABI of the attention step (include/openmini_attn.h, and the decode call of
// include/openmini_kv_i8.h): argument checks and kernel
// dispatch.  Host code only; every failure returns a status and leaves a message.
#include <new>

#include "attn_check.hpp"

using namespace attn;

namespace {

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

bool decode_sizes(int q_heads, int kv_heads, int head_dim, int* head_tiles) {
    if (kv_heads < 1 || q_heads < kv_heads || q_heads > 1024 || q_heads % kv_heads ||
        !decode_dim(head_dim))
        return false;
    const int group = q_heads / kv_heads;
    *head_tiles = (group + attn::kHeadTile - 1) / attn::kHeadTile;
    return true;
}

// Both decode calls: on 8-bit integers with the blocks' scales (i8), or on the other caches.
int decode(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales, const openmini_attn_args_t* p, void* stream,
           bool i8) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    attn::DecodeI8Args a = {};
    TRY(i8 ? check_cache_i8(cache, scales, &a.cache, &a.scales) : check_cache(cache, &a.cache));
    if (!half_type(p->q_dtype)) return unsupported("q", p->q_dtype);
    const bool f8 = i8 || cache->dtype == OPENMINI_ATTN_F8_E4M3;  // an element is a byte
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
    const int sub = i8 ? attn::decode_subtiles_i8(cache->head_dim) : attn::decode_subtiles(cache->head_dim, f8), tile = 32 * sub;
    const int64_t tiles = p->rows * (max_len / tile + 2);  // of the call at most
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
    const int64_t keys = max_len < (int64_t)a.window ? max_len : (int64_t)a.window;
    a.stream = head_tiles == 1 && p->rows <= p->requests &&
               attn::decode_streams(c, cache->kv_heads, cache->head_dim, f8, p->rows * keys);
    // a window's first tile need not begin with it
    const int64_t most = (keys + tile - 1) / tile + (keys < max_len), pairs = p->rows * cache->kv_heads * head_tiles;
    a.whole = attn::decode_whole(most, pairs);
    const int64_t units = (int64_t)cache->kv_heads * head_tiles;
    a.uncut = i8 ? attn::decode_uncut_i8(most, p->rows, units, shares, cache->head_dim)
                 : attn::decode_uncut(most, p->rows, units, shares, cache->head_dim, f8);
    if (a.uncut) a.launch_shares = p->rows < (int64_t)shares ? (uint32_t)p->rows : shares;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool bf16 = p->q_dtype == OPENMINI_ATTN_BF16;
    hipError_t e = i8     ? (bf16 ? attn::launch_decode_i8_bf16 : attn::launch_decode_i8_f16)(a, cache->head_dim, s)
                   : bf16 ? attn::launch_decode_bf16(a, cache->head_dim, f8, s)
                          : attn::launch_decode_f16(a, cache->head_dim, f8, s);
    if (e == hipSuccess && !a.whole && !a.uncut && a.launch_shares > 1)
        e = attn::launch_join(a, cache->head_dim, p->out_dtype, s);
    return launched(e, "attention launch");
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
    TRY(check_append(rope, cache, p));
    a.k_over = 1.0f / cache->k_scale;
    a.v_over = 1.0f / cache->v_scale;
    if (!std::isfinite(a.k_over) || !std::isfinite(a.v_over))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "cache scales %g, %g: below 2^-128 they have no reciprocal", cache->k_scale,
                    cache->v_scale);
    if (p->tokens == 0) return ok();
    set_append(a, rope, cache, p);
    return launched(attn::launch_rope(a, cache->head_dim, static_cast<hipStream_t>(stream)), "rope append launch");
}

size_t openmini_attn_workspace_bytes(int q_heads, int kv_heads, int head_dim) {
    int head_tiles = 0;
    if (!decode_sizes(q_heads, kv_heads, head_dim, &head_tiles)) return 0;
    return workspace(q_heads, kv_heads, head_tiles, head_dim).bytes;
}

int openmini_attn_decode(const openmini_kv_cache_t* cache, const openmini_attn_args_t* p, void* stream) {
    return decode(cache, nullptr, p, stream, false);
}

int openmini_attn_decode_i8(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales, const openmini_attn_args_t* p,
                            void* stream) {
    return decode(cache, scales, p, stream, true);
}

}  // extern "C"
