/*
 * openmini_attn.h -- C ABI of the attention step between a layer's q / k / v projections
 * and its output projection, on MI355X (gfx950): pages and slots for a step's tokens,
 * rotary positions, the key-value cache write, and the attention of single query tokens
 * over the paged cache.
 *
 * Part of libopenmini_qmm.so.  Conventions are those of openmini_qmm.h, whose status
 * codes these calls return: no call aborts, a failing one leaves its message in
 * openmini_qmm_last_error() and goes to the log callback; d_* are device pointers that
 * stay valid until the stream reaches the call; `stream` NULL is the null stream.  Every
 * call only enqueues work (one kernel launch, attention at most two; no allocation, no copy, no
 * synchronisation), so a stream capture may hold them.
 *
 * All numbers of tokens, slots and pages are int32 on the device.  What a call reads from
 * device arrays (lengths, tables, slots) is checked in its kernel against the sizes given
 * by the host: a length past the table counts as the table's, a page or slot outside the
 * cache is neither read nor written.  Sizes, strides and alignment are checked on the host.
 */
#pragma once

#include "openmini_qmm.h"

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* Element types of activations and caches. */
typedef enum {
    OPENMINI_ATTN_F32 = 0,
    OPENMINI_ATTN_F16 = 1,
    OPENMINI_ATTN_BF16 = 2,
    OPENMINI_ATTN_F8_E4M3 = 3 /* OCP e4m3 (no infinities, largest value 448); caches only */
} openmini_attn_dtype_t;

/* ---- the paged cache ----------------------------------------------------------------
 * Keys and values of one layer, in the caller's memory: n_pages pages of page_size tokens.
 * Element (page p, token t of the page, head h, dimension i) of d_k, and of d_v alike, is
 * at p * page_stride + t * token_stride + h * head_stride + i, in elements.  So
 * [pages][page_size][kv_heads][head_dim] and [pages][kv_heads][page_size][head_dim] are
 * both caches, and keys and values may be interleaved in one array.  A stored element
 * stands for itself times k_scale (v_scale), which are 1 for the 16-bit types as a rule.
 * Pointers and the three strides are multiples of 16 bytes; n_pages * page_size is at most
 * 2^31 - 1.  Slot s of the cache is token s % page_size of page s / page_size. */
typedef struct {
    void* d_k;
    void* d_v;
    int32_t dtype; /* F16, BF16 or F8_E4M3 */
    int32_t kv_heads;
    int32_t head_dim;
    int32_t page_size;
    int64_t n_pages;
    int64_t page_stride;
    int64_t token_stride;
    int64_t head_stride;
    float k_scale;
    float v_scale;
} openmini_kv_cache_t;

/* ---- pages and slots of a step ------------------------------------------------------
 * Request r holds d_cached[r] tokens and adds d_new[r] (negative values count as 0).  It
 * needs ceil((cached + new) / page_size) - ceil(cached / page_size) pages more, which it
 * takes from d_free in request order, starting at *d_head (NULL: at 0), into its table:
 * d_tables[r * table_stride + i] is the page of its tokens i * page_size on.  Nothing else
 * of the tables is written.  A request is refused, and takes nothing, if its tokens would
 * not fit max_pages pages, or if it needs pages and the free list has fewer than it and all
 * requests before it need (those too long for the table apart).  So the first request that is
 * short of pages refuses all behind it that need any, also where what is left would do for
 * them: the order of requests is that in which they are served, and a server that wants its
 * decoding requests to go on puts them before the prompts.  Outputs:
 *   d_starts[requests + 1]  first token of each request in the step, and the token count
 *   d_lens[requests]        cached + new (refused: cached)
 *   for token j < max_tokens, request after request (-1, -1, -1, 0 past the last):
 *   d_rows[j]               its request
 *   d_positions[j]          its position in the request
 *   d_slots[j]              its cache slot (refused: -1)
 *   d_row_lens[j]           position + 1, the keys that a causal query of it sees (refused: 0)
 *   d_counts[4]             tokens, pages taken, requests refused, the next *d_head
 * A step of more than max_tokens tokens keeps its first max_tokens (counts[0] tells).  No
 * output may share memory with an input: d_head is not &d_counts[3] of the same call (copy it
 * on the stream, or let the steps take turns with two counts).  1 <= requests <= 4096. */
typedef struct {
    const int32_t* d_cached;
    const int32_t* d_new;
    int64_t requests;
    const int32_t* d_free;
    int64_t n_free;
    const int32_t* d_head; /* NULL: 0 */
    int32_t* d_tables;
    int64_t table_stride;
    int64_t max_pages; /* columns of a table, at most table_stride */
    int64_t page_size;
    int64_t max_tokens;
    int32_t* d_starts;
    int32_t* d_lens;
    int32_t* d_rows;
    int32_t* d_positions;
    int32_t* d_slots;
    int32_t* d_row_lens;
    int32_t* d_counts;
} openmini_kv_plan_args_t;

int openmini_kv_plan(const openmini_kv_plan_args_t* args, void* stream);

/* ---- rotary positions ---------------------------------------------------------------
 * Pair i of a head's first 2 * pairs dimensions turns by position[axis[i]] * inv_freq[i]
 * radians and is multiplied by `scale`; the rest of the head passes through unscaled.
 * With one axis that is text; with three (time, height, width), images and video.
 * inv_freq and axis are host arrays of `pairs` entries (axis NULL: all 0); the handle
 * keeps them on the current device, the frequencies as 64-bit fractions of a revolution,
 * so that an angle is reduced exactly whatever the position.  Pairs are dimensions
 * (i, i + pairs) or, with `adjacent`, (2 i, 2 i + 1).  pairs: a multiple of 4, at most 128;
 * axes: 1 to 8. */
typedef struct openmini_rope openmini_rope_t;

int openmini_rope_create(const double* inv_freq, const int32_t* axis, int pairs, int axes, int adjacent, float scale,
                         openmini_rope_t** out_rope);
/* The caller has waited for the calls that use it. */
void openmini_rope_free(openmini_rope_t* rope);

/* y = x with its heads rotated, [tokens][heads][head_dim] each, `x_stride` (`y_stride`)
 * elements from a token to the next.  inverse != 0 turns the other way: the gradient of x
 * from that of y.  Position of token j on axis a: d_positions[a * position_stride + j].
 * x and y are F32, F16 or BF16; they may be the same memory where type and stride are the
 * same.  head_dim: a multiple of 8, at most 512; pointers 16-byte aligned and strides
 * multiples of 16 bytes. */
typedef struct {
    const void* d_x;
    void* d_y;
    int64_t x_stride;
    int64_t y_stride;
    int32_t x_dtype;
    int32_t y_dtype;
    int64_t tokens;
    int32_t heads;
    int32_t head_dim;
    int32_t inverse;
    const int32_t* d_positions;
    int64_t position_stride;
} openmini_rope_args_t;

int openmini_rope_apply(const openmini_rope_t* rope, const openmini_rope_args_t* args, void* stream);

/* One step of a layer: q rotated to d_q_out; k rotated, and v as it is, each times the
 * reciprocal of its scale (which is above 2^-128), rounded to the cache's type (F8: to the nearest even, values past +-448 to +-448,
 * NaN stays) and written at the tokens' slots.  A token whose slot is negative or past the
 * cache writes q alone.  Two tokens with one slot: either is written.  d_q, d_k and d_v are
 * [tokens][heads | kv_heads][head_dim] of one type, token strides in elements (slices of
 * one fused projection will do).  q_out is F16 or BF16 and none of the inputs. */
typedef struct {
    const void* d_q;
    const void* d_k;
    const void* d_v;
    int64_t q_stride;
    int64_t k_stride;
    int64_t v_stride;
    void* d_q_out;
    int64_t q_out_stride;
    int32_t in_dtype;    /* F32, F16 or BF16 */
    int32_t q_out_dtype; /* F16 or BF16 */
    int64_t tokens;
    int32_t q_heads;
    const int32_t* d_positions;
    int64_t position_stride;
    const int32_t* d_slots;
} openmini_rope_append_args_t;

int openmini_rope_append(const openmini_rope_t* rope, const openmini_kv_cache_t* cache,
                         const openmini_rope_append_args_t* args, void* stream);

/* ---- attention of single query tokens -----------------------------------------------
 * Row j is one query token of request d_rows[j] (NULL: of request j) that sees the
 * request's keys 0 .. d_lens[j] - 1, or with window > 0 the last `window` of them:
 *   s_i = scale * q . k_i,  out = sum_i softmax(s)_i v_i,  lse = log sum_i exp(s_i).
 * Query head h reads key head h / (q_heads / kv_heads).  A row that sees no key, or whose
 * request is outside [0, requests), is 0 with lse -inf; keys on pages outside the cache are
 * not seen.  What the cache holds past a row's keys does not matter (NaN included).  Among
 * them, a key whose score is -inf has no weight, and a row with no other is empty too; a score
 * of +inf or NaN makes its head NaN.  A value that is NaN makes its dimension of all heads
 * that read it NaN, one that is infinite makes it infinite or NaN (a probability is several
 * factors, some of them 0 or below).  d_out, d_lse and d_work share no memory with the inputs.
 *
 * Types: q F16 or BF16 and the cache the same type, or F8_E4M3, which is converted to q's
 * (exactly); out q's type or F32.  Products are of 16-bit operands with 32-bit sums; the
 * probabilities enter the second product as the sum of three bf16 parts, which hold 24 bits of
 * them, or on an F16 cache of fp16 parts, which hold 22 bits of them down to 2^-57 of a row's
 * largest and all of them to 2^-79 of it.  head_dim: 64, 96, 128, 192 or 256; page_size: a multiple
 * of 8; q_heads: a multiple of kv_heads, at most 1024.
 *
 * Long rows are cut into parts that separate waves take, and a second launch joins a row's
 * parts in their order; where the tables and the window leave only short rows, a workgroup
 * takes a row, or a wave several, and there is no second launch (so max_pages is best no more than the call's
 * longest row needs; table_stride is free).  How rows are cut depends on all lengths of the
 * call and on max_pages, so the last bits of a row may differ between calls with other rows
 * beside it; equal calls give equal bits.  d_work: openmini_attn_workspace_bytes bytes,
 * 256-byte aligned, of any content; two calls that share it must not overlap in time. */
typedef struct {
    const void* d_q;
    int64_t q_stride; /* elements from a row to the next; a row is [q_heads][head_dim] */
    void* d_out;
    int64_t out_stride;
    float* d_lse; /* [rows][q_heads], or NULL */
    int32_t q_dtype;
    int32_t out_dtype;
    int32_t q_heads;
    float scale;
    int64_t window; /* 0: all keys */
    int64_t rows;
    const int32_t* d_lens;
    const int32_t* d_rows; /* NULL: row j reads table j */
    const int32_t* d_tables;
    int64_t table_stride;
    int64_t max_pages; /* columns of a table that hold pages, at most table_stride */
    int64_t requests;  /* tables */
    void* d_work;
    size_t work_bytes;
} openmini_attn_args_t;

/* Bytes of d_work for calls of any number of rows; 0 for sizes that openmini_attn_decode
 * does not take.  Calls of several sizes may take turns with the largest of theirs. */
size_t openmini_attn_workspace_bytes(int q_heads, int kv_heads, int head_dim);
int openmini_attn_decode(const openmini_kv_cache_t* cache, const openmini_attn_args_t* args, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
