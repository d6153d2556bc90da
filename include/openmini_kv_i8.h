/*
 * openmini_kv_i8.h -- C ABI of key-value caches in 8-bit integers with a scale for each
 * block of tokens and head, on MI355X (gfx950): the quantising cache write, attention of
 * single query tokens, and two calls that take every cache: attention of runs of query
 * tokens (prompts) and reading a cache back.
 *
 * Part of libopenmini_qmm.so.  Conventions, the paged cache and its other calls are those of
 * openmini_attn.h: no call aborts, every call only enqueues work on `stream`, and what
 * device arrays say (lengths, tables, slots, starts) is checked in the kernels.
 */
#pragma once

#include "openmini_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* ---- caches in 8-bit integers ---------------------------------------------------------
 * An openmini_kv_cache_t of this dtype (k_scale and v_scale 1; its strides multiples of 16
 * elements, which are bytes here) holds codes of -127 to 127;
 * an element stands for its code times the scale of its block: `block` tokens of a page
 * (8, 16 or 32; page_size is a multiple of it) of one head.  The scale of block b of page p
 * and head h is element p * page_stride + b * block_stride + h * head_stride of d_k, and of
 * d_v alike.  No two scales share an element.  A scale is positive (0 stands for a block of
 * zeros).  To attention a block whose scale is NaN or infinite is NaN as a whole;
 * openmini_kv_read gives the products (under an infinite scale infinities, NaN for codes of 0). */
#define OPENMINI_ATTN_I8 4

typedef struct {
    float* d_k;
    float* d_v;
    int32_t block;
    int64_t page_stride;
    int64_t block_stride;
    int64_t head_stride;
} openmini_kv_scales_t;

/* openmini_rope_append on a cache of 8-bit integers.  The call's tokens of one block follow
 * each other in the arrays, their slots one apart (as openmini_kv_plan lays them out; if they
 * do not, what the block holds afterwards is unspecified).  With `first` the place of the
 * first of them in the block, the tokens before it are held already and those behind it are
 * not.  For a block and head, a = max |x| of its new elements (k after its turn), and in fp32, each
 * operation rounded (1/127 is one number, and so is 1 / s', which elements are multiplied by):
 *   n = max(a * (1/127), 2^-40)
 *   s' = n where first = 0; else the old s where s >= n; else max(n, 1.25 * s)
 *   new codes: x * (1 / s') rounded to the nearest even;  held codes c: c * (s / s') likewise.
 * So all roundings of an element add up to at most 2.5 s', whatever the order in which a
 * block fills.  An element that is NaN or infinite makes s' NaN, until a call starts the block
 * with first = 0.  head_dim is at most 256.  One call at a time writes a block: two requests that share a block which
 * is not full each need a copy of it before they go on.  Keys and values share no element, nor do their scales, nor
 * two slots; interleaved in one array they may be. */
int openmini_rope_append_i8(const openmini_rope_t* rope, const openmini_kv_cache_t* cache,
                            const openmini_kv_scales_t* scales, const openmini_rope_append_args_t* args, void* stream);

/* openmini_attn_decode on a cache of 8-bit integers, with the same workspace: products of
 * the codes, which are exact in 16 bits; the scales multiply fp32 scores and probabilities.  q is
 * F16 or BF16, out q's type or F32.  A block of keys whose scale is NaN or infinite makes the
 * heads that see it NaN, a block of values their outputs. */
int openmini_attn_decode_i8(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales,
                            const openmini_attn_args_t* args, void* stream);

/* ---- reading a cache back -------------------------------------------------------------
 * Row d_starts[r] + i of d_k_out and d_v_out, up to row d_starts[r + 1] - 1, is token
 * d_first[r] + i of request r (d_first NULL: from token 0 on), whose pages are
 * d_tables[r * table_stride + ...]: [kv_heads][head_dim] elements of type out_dtype (F32, F16 or
 * BF16), each rounded once; `k_stride` (`v_stride`) elements from a row to the next.  A token
 * past the table, before 0 or on a page outside the cache reads as zeros.  Rows of no request are
 * left as they were, and so are those from `tokens` on.  d_starts does not decrease.  Either
 * output may be NULL; rows of both may take turns in one array (of one stride), but an output, from its
 * first row to its last, shares no memory with what the call reads.  Caches of every type; `scales` is NULL
 * but for 8-bit integers.
 * head_dim: a multiple of 8, at most 512; tokens: at most 2^26; requests: at most 2^20. */
typedef struct {
    const int32_t* d_tables;
    int64_t table_stride;
    int64_t max_pages;
    int64_t requests;
    const int32_t* d_starts; /* [requests + 1] */
    const int32_t* d_first;  /* [requests], or NULL */
    int64_t tokens;          /* rows of the outputs */
    void* d_k_out;
    void* d_v_out;
    int64_t k_stride;
    int64_t v_stride;
    int32_t out_dtype;
} openmini_kv_read_args_t;

int openmini_kv_read(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales,
                     const openmini_kv_read_args_t* args, void* stream);

/* ---- attention of runs of query tokens ------------------------------------------------
 * Rows d_starts[r] to d_starts[r + 1] - 1 are query tokens of request r, and row j of them sees
 * the request's keys 0 .. d_lens[j] - 1, or with window > 0 the last `window` of them (a prompt's
 * tokens, the last of which sees all keys: openmini_kv_plan's starts and row_lens):
 *   s_i = scale * q . k_i,  out = sum_i softmax(s)_i v_i,  lse = log sum_i exp(s_i).
 * What openmini_attn_decode says of heads, of rows without keys, of pages outside the cache,
 * of infinite and NaN scores and values, and of what lies past a row's keys holds here too, but
 * an infinite value may make its dimension NaN, and a block of values whose scale is NaN or
 * infinite makes lse NaN too.  Rows of no request are left as they were.  d_starts does not decrease.
 * Keys and values are read once for a tile of query tokens and heads, so a call of many rows
 * to a request takes the time of its products.
 *
 * Types: q F16 or BF16; the cache of q's type (`scales` NULL), F8_E4M3 (NULL) or I8; out q's
 * type or F32.  Products are of 16-bit operands with 32-bit sums.  With 16-bit outputs a
 * probability is rounded once to 16 bits: bf16 on BF16 caches; else fp16, which holds 11 bits of
 * it down to 2^-25 of a row's largest (values' scales included) and less below, nothing from
 * 2^-36 on.  With F32 outputs it enters as the sum of three bf16 parts, or on F16 caches as in
 * openmini_attn_decode.  Sums, maxima and lse are fp32.  head_dim: 64, 96, 128, 192 or 256;
 * page_size: a multiple of 8; q_heads: a multiple of kv_heads, at most 1024; requests: at most
 * 2^20.  A scale of 8-bit values below 2^-60 counts as 2^-60, one above 2^126 as infinite; those
 * of a row's blocks are within 2^100 of each other (past that the keys of the least lose weight).
 *
 * Where the tiles are few for the chip, and the table long, several workgroups take parts
 * of a tile's keys and a second launch joins them in order: by the sizes of the call, so equal
 * calls give equal bits.  d_work: openmini_attn_prompt_workspace_bytes bytes, 256-byte aligned,
 * of any content; two calls that share it must not overlap in time. */
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
    const int32_t* d_lens;   /* [rows] */
    const int32_t* d_starts; /* [requests + 1] */
    const int32_t* d_tables;
    int64_t table_stride;
    int64_t max_pages;
    int64_t requests;
    void* d_work;
    size_t work_bytes;
} openmini_attn_prompt_args_t;

/* Bytes of d_work for calls of any number of rows; 0 for sizes that the call does not take. */
size_t openmini_attn_prompt_workspace_bytes(int q_heads, int kv_heads, int head_dim);
int openmini_attn_prompt(const openmini_kv_cache_t* cache, const openmini_kv_scales_t* scales,
                         const openmini_attn_prompt_args_t* args, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
