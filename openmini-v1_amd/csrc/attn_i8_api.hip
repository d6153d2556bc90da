// C ABI of include/openmini_kv_i8.h but for its decode call (attn_api.hip): argument checks and
// kernel dispatch.  Host code only; every failure returns a status and leaves a message.
#include "attn_check.hpp"

using namespace attn;

namespace {

constexpr int64_t kMaxRuns = (int64_t)1 << 20;
constexpr int64_t kMaxThreads = (int64_t)UINT32_MAX;  // of a launch
constexpr int64_t kMaxI64 = INT64_MAX;

bool prompt_sizes(int q_heads, int kv_heads, int head_dim) {
    return kv_heads >= 1 && q_heads >= kv_heads && q_heads <= 1024 && q_heads % kv_heads == 0 && decode_dim(head_dim);
}

// The workspace: the parts' maxima and sums, then their accumulators.
size_t ml_bytes(int head_dim) { return (size_t)kPromptParts * prompt_rows(head_dim) * 8; }

// Workgroups read at their own time what others may have written already: an output, from its first
// row to its last, shares nothing with what the call reads, nor its rows with the other's.
int check_read_memory(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales, const openmini_kv_read_args_t* p, int size,
                      int64_t row_bytes) {
    const Box<4> elements = cache_bytes(cache, size_of(cache->dtype));
    struct {
        const void* at;
        int64_t stride;
    } out[] = {{p->d_k_out, p->k_stride * size}, {p->d_v_out, p->v_stride * size}};
    const struct {
        const char* name;
        const void* at;
        int64_t bytes;
    } in[] = {{"d_tables", p->d_tables, 4 * ((p->requests - 1) * p->table_stride + p->max_pages)},
              {"d_starts", p->d_starts, 4 * (p->requests + 1)},
              {"d_first", p->d_first, 4 * p->requests}};
    int64_t bytes[2] = {0, 0};
    for (int i = 0; i < 2; ++i) {
        if (!out[i].at) continue;  // nor is its stride looked at
        // saturated: no memory is as large
        bytes[i] = p->tokens - 1 > kMaxI64 / 4 / out[i].stride ? kMaxI64 / 4 : (p->tokens - 1) * out[i].stride + row_bytes;
        const char* with = nullptr;
        for (const auto& x : in)
            if (x.at && bytes_apart(out[i].at, x.at) < x.bytes && bytes_apart(x.at, out[i].at) < bytes[i]) with = x.name;
        for (const void* at : {cache->d_k, cache->d_v}) {
            const int64_t from = bytes_apart(out[i].at, at);
            if (elements.meets(from, from + bytes[i])) with = "the cache";
        }
        if (scales)
            for (const void* at : {scales->d_k, scales->d_v}) {
                const int64_t from = bytes_apart(out[i].at, at);
                if (scale_bytes(cache, scales).meets(from, from + bytes[i])) with = "the scales";
            }
        if (with) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%s and %s share memory", i ? "d_v_out" : "d_k_out", with);
    }
    if (!out[0].at || !out[1].at) return OPENMINI_QMM_OK;
    const int64_t apart = bytes_apart(out[1].at, out[0].at);
    const Axis axes[] = {{1, row_bytes}, {out[0].stride, p->tokens}};
    if (out[0].stride == out[1].stride ? Box<2>(axes).meets_itself(apart) : apart < bytes[0] && -apart < bytes[1])
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_k_out and d_v_out share memory");
    return OPENMINI_QMM_OK;
}

}  // namespace

extern "C" {

int openmini_rope_append_i8(const openmini_rope_t* rope, const openmini_kv_cache_t* cache,
                            const openmini_kv_scales_t* scales, const openmini_rope_append_args_t* p, void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    if (!rope) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null rope handle");
    AppendI8Args a = {};
    TRY(check_cache_i8(cache, scales, &a.r.cache, &a.scales));
    // Keys and values are written by workgroups of their own, at their own time.
    const Box<4> codes = cache_bytes(cache, 1), of_blocks = scale_bytes(cache, scales);
    if (!codes.nested)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "cache strides %lld, %lld, %lld: two slots share memory", (long long)cache->page_stride,
                    (long long)cache->token_stride, (long long)cache->head_stride);
    if (codes.meets_itself(bytes_apart(cache->d_v, cache->d_k)))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "the cache's d_k and d_v share memory");
    if (of_blocks.meets_itself(bytes_apart(scales->d_v, scales->d_k)))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "the scales' d_k and d_v share memory");
    TRY(check_rope(rope));
    TRY(check_append(rope, cache, p));
    if (cache->head_dim > kMaxI8Dim)
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "head_dim = %d on a cache of 8-bit integers: at most %d", cache->head_dim, kMaxI8Dim);
    const int64_t groups = p->tokens * ((p->q_heads * (cache->head_dim / 8) + 255) / 256) + 2 * (p->tokens / 16 + 1) * cache->kv_heads;
    if (groups * 256 > kMaxThreads)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%lld tokens are too many for one call", (long long)p->tokens);
    if (p->tokens == 0) return ok();
    set_append(a.r, rope, cache, p);
    a.r.per_token = FastDiv((uint32_t)(p->q_heads * (cache->head_dim / 8)));
    return launched(launch_append_i8(a, cache->head_dim, static_cast<hipStream_t>(stream)), "rope append launch");
}

int openmini_kv_read(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales, const openmini_kv_read_args_t* p,
                     void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    ReadArgs a = {};
    TRY(check_any_cache(cache, scales, &a.cache, &a.scales));
    if (!dense_type(p->out_dtype)) return unsupported("k_out, v_out", p->out_dtype);
    TRY(check_range("requests", p->requests, 1, kMaxRuns));
    TRY(check_range("tokens", p->tokens, 0, (int64_t)1 << 26));
    TRY(check_range("max_pages", p->max_pages, 1, kMaxI32));
    TRY(check_range("table_stride", p->table_stride, p->max_pages, (int64_t)1 << 40));
    TRY(check_pointer("d_tables", p->d_tables, 4));
    TRY(check_pointer("d_starts", p->d_starts, 4));
    if (p->d_first) TRY(check_pointer("d_first", p->d_first, 4));
    if (!p->d_k_out && !p->d_v_out) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_k_out and d_v_out are both null");
    const int size = size_of(p->out_dtype);
    const int64_t row = (int64_t)cache->kv_heads * cache->head_dim;
    if (p->d_k_out) {
        TRY(check_pointer("d_k_out", p->d_k_out, 16));
        TRY(check_stride("k_stride", p->k_stride, row, size));
    }
    if (p->d_v_out) {
        TRY(check_pointer("d_v_out", p->d_v_out, 16));
        TRY(check_stride("v_stride", p->v_stride, row, size));
    }
    if (p->tokens == 0) return ok();
    if (p->d_k_out == p->d_v_out) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_k_out is d_v_out");
    for (const void* out : {p->d_k_out, p->d_v_out})
        if (out && (out == cache->d_k || out == cache->d_v))
            return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "an output is the cache");
    TRY(check_read_memory(cache, scales, p, size, row * size));
    TRY(qmm::current_device(nullptr));
    const int64_t held = p->max_pages * cache->page_size;
    a.tables = p->d_tables;
    a.starts = p->d_starts;
    a.first = p->d_first;
    a.table_stride = p->table_stride;
    a.requests = (uint32_t)p->requests;
    a.max_len = (uint32_t)(held < kMaxI32 ? held : kMaxI32);
    a.tokens = p->tokens;
    a.k_out = static_cast<uint8_t*>(p->d_k_out);
    a.v_out = static_cast<uint8_t*>(p->d_v_out);
    a.k_stride = p->k_stride * size;
    a.v_stride = p->v_stride * size;
    a.kv_heads = cache->kv_heads;
    a.out_dtype = p->out_dtype;
    a.cache_dtype = cache->dtype;
    a.per_head = FastDiv((uint32_t)cache->head_dim / 8);
    a.per_token = FastDiv((uint32_t)(cache->kv_heads * (cache->head_dim / 8)));
    return launched(launch_read(a, static_cast<hipStream_t>(stream)), "cache read launch");
}

size_t openmini_attn_prompt_workspace_bytes(int q_heads, int kv_heads, int head_dim) {
    if (!prompt_sizes(q_heads, kv_heads, head_dim)) return 0;
    return ml_bytes(head_dim) * (1 + (size_t)head_dim / 2);
}

int openmini_attn_prompt(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales,
                         const openmini_attn_prompt_args_t* p, void* stream) {
    if (!p) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "null arguments");
    PromptArgs a = {};
    TRY(check_any_cache(cache, scales, &a.cache, &a.scales));
    if (!half_type(p->q_dtype)) return unsupported("q", p->q_dtype);
    if (half_type(cache->dtype) && cache->dtype != p->q_dtype)
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "q of type %d on a cache of type %d", p->q_dtype, cache->dtype);
    if (p->out_dtype != p->q_dtype && p->out_dtype != OPENMINI_ATTN_F32) return unsupported("out", p->out_dtype);
    if (!decode_dim(cache->head_dim))
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "head_dim = %d (64, 96, 128, 192 and 256 are taken)", cache->head_dim);
    if (cache->page_size % 8)
        return fail(OPENMINI_QMM_ERR_UNSUPPORTED, "page_size = %d is not a multiple of 8", cache->page_size);
    if (!prompt_sizes(p->q_heads, cache->kv_heads, cache->head_dim))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "q_heads = %d for kv_heads = %d: a multiple, at most 1024", p->q_heads,
                    cache->kv_heads);
    TRY(check_range("rows", p->rows, 0, kMaxRows));
    TRY(check_range("requests", p->requests, 1, kMaxRuns));
    TRY(check_pointer("d_q", p->d_q, 16));
    TRY(check_pointer("d_out", p->d_out, 16));
    TRY(check_pointer("d_lens", p->d_lens, 4));
    TRY(check_pointer("d_starts", p->d_starts, 4));
    TRY(check_pointer("d_tables", p->d_tables, 4));
    if (p->d_lse) TRY(check_pointer("d_lse", p->d_lse, 4));
    if (p->d_out == p->d_q) return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_out is d_q");
    if (p->d_lse && ((const void*)p->d_lse == p->d_out || (const void*)p->d_lse == p->d_q))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "d_lse is d_out or d_q");
    const int64_t row = (int64_t)p->q_heads * cache->head_dim;
    const int out_size = size_of(p->out_dtype);
    TRY(check_stride("q_stride", p->q_stride, row, 2));
    TRY(check_stride("out_stride", p->out_stride, row, out_size));
    const float scale = (float)((double)p->scale * cache->k_scale * 1.44269504088896340736);
    if (!std::isfinite(scale))
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "scale %g (times the keys' %g and log2(e)) is not finite", p->scale, cache->k_scale);
    TRY(check_range("window", p->window, 0, INT64_MAX));
    TRY(check_range("max_pages", p->max_pages, 1, kMaxI32));
    TRY(check_range("table_stride", p->table_stride, p->max_pages, (int64_t)1 << 40));
    if (p->rows == 0) return ok();
    const size_t ml = ml_bytes(cache->head_dim), need = openmini_attn_prompt_workspace_bytes(p->q_heads, cache->kv_heads, cache->head_dim);
    TRY(check_pointer("d_work", p->d_work, 256));
    if (p->work_bytes < need)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "workspace of %zu bytes, %zu are needed", p->work_bytes, need);
    const int64_t held = p->max_pages * cache->page_size, max_len = held < kMostKeys ? held : kMostKeys;
    a.group = p->q_heads / cache->kv_heads;
    // keys that a tile sees at most: all, or its rows' windows (a run's lengths rise by one)
    const int64_t seen = p->window && p->window < max_len - 256 ? p->window + 256 : max_len;
    const PromptShape shape = prompt_shape(cache->head_dim, p->rows, p->requests, cache->kv_heads, a.group, seen);
    if (shape.wgs() * 64 * shape.waves > kMaxThreads)
        return fail(OPENMINI_QMM_ERR_INVALID_PARAM, "%lld rows of %lld requests are too many for one call", (long long)p->rows,
                    (long long)p->requests);
    TRY(qmm::current_device(nullptr));
    a.q = static_cast<const uint8_t*>(p->d_q);
    a.out = static_cast<uint8_t*>(p->d_out);
    a.lse = p->d_lse;
    a.lens = p->d_lens;
    a.starts = p->d_starts;
    a.tables = p->d_tables;
    a.q_stride = p->q_stride * 2;
    a.out_stride = p->out_stride * out_size;
    a.table_stride = p->table_stride;
    a.rows = (uint32_t)p->rows;
    a.requests = (uint32_t)p->requests;
    a.max_len = (uint32_t)max_len;
    a.window = p->window && p->window < max_len ? (uint32_t)p->window : (uint32_t)max_len;
    a.q_heads = p->q_heads;
    a.by_tokens = FastDiv((uint32_t)shape.tokens);
    a.by_heads = FastDiv((uint32_t)shape.heads);
    a.by_units = FastDiv((uint32_t)shape.units);
    a.by_head_tiles = FastDiv((uint32_t)shape.head_tiles);
    a.negative = scale < 0;
    // a score of -inf (a key that is not seen) stays one under a scale of zero
    a.scale = std::fmax(std::fabs(scale), 1e-37f);
    a.waves = shape.waves;
    a.tiles = (uint32_t)shape.tiles;
    a.splits = (uint32_t)shape.splits;
    a.part_ml = static_cast<float2*>(p->d_work);
    a.part_acc = reinterpret_cast<float*>(static_cast<uint8_t*>(p->d_work) + ml);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e = (p->q_dtype == OPENMINI_ATTN_BF16 ? launch_prompt_bf16 : launch_prompt_f16)(
        a, cache->head_dim, cache->dtype, p->out_dtype == OPENMINI_ATTN_F32, s);
    if (e == hipSuccess && a.splits > 1) e = launch_prompt_join(a, cache->head_dim, p->out_dtype, s);
    return launched(e, "prompt attention launch");
}

}  // extern "C"
