// Declarations shared by the attention step's C ABI (attn_api.hip) and its kernels
// (attn_plan.hip, attn_rope.hip, attn_decode.hpp).
#pragma once

#include "attn_decode_shape.hpp"
#include "attn_prompt_shape.hpp"
#include "qmm_internal.hpp"

#include "../../include/openmini_kv_i8.h"

namespace attn {

// n / d for 0 <= n < 2^31 by one multiplication: with l = ceil(log2 d) >= 1 and
// m = ceil(2^(31 + l) / d) < 2^32, m d exceeds 2^(31 + l) by less than d <= 2^l, so
// floor(n m / 2^(31 + l)) = floor(n / d) while n < 2^31.  d = 1 is m = 0.
struct FastDiv {
    uint32_t d = 1, m = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        uint32_t l = 0;
        while (((uint64_t)1 << l) < div) ++l;
        if (l == 0) return;
        shift = l - 1;
        m = (uint32_t)((((uint64_t)1 << (31 + l)) + div - 1) / div);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return m ? __umulhi(n, m) >> shift : n; }
    __device__ __forceinline__ uint32_t div_by_many(uint32_t n) const { return __umulhi(n, m) >> shift; }  // d > 1
};

// A cache as the kernels see it: strides in bytes.
struct Cache {
    uint8_t* k;
    uint8_t* v;
    int64_t page_stride, token_stride, head_stride;
    uint32_t n_pages, slots;  // slots = n_pages * page_size
    FastDiv page;
    float k_scale, v_scale;
};

// The scales of a cache of 8-bit integers: strides in elements, tokens to a block 2^shift.
struct Scales {
    float *k, *v;
    int64_t page_stride, block_stride, head_stride;
    uint32_t shift;
};

// ---- attn_plan.hip -------------------------------------------------------------------
constexpr int kMaxPlanRequests = 4096;  // three words a request in a workgroup's LDS

struct PlanArgs {
    const int32_t *cached, *fresh, *free, *head;
    int32_t *tables, *starts, *lens, *rows, *positions, *slots, *row_lens, *counts;
    int64_t table_stride;
    uint32_t requests, n_free, max_held, max_tokens;  // max_held = max_pages * page_size
    FastDiv page;
};
hipError_t launch_plan(const PlanArgs& a, hipStream_t s);

// ---- attn_rope.hip -------------------------------------------------------------------
constexpr int kMaxPairs = 128;
constexpr int kMaxAxes = 8;

struct RopePair {
    uint64_t step;  // revolutions a position, as a fraction of 2^64
    int32_t axis;
    int32_t unused;
};

struct Rope {
    RopePair* pairs;  // device
    int32_t n_pairs, axes, adjacent;
    float scale;
};

struct RopeArgs {
    // tokens x (heads + 2 kv_heads) heads: the first `heads` turned into y, then (append)
    // kv_heads of k turned into the cache and kv_heads of v written to it
    const uint8_t *x, *k, *v;
    int64_t x_stride, k_stride, v_stride, y_stride;  // bytes a token
    uint8_t* y;
    const int32_t* positions;
    int64_t position_stride;
    const int32_t* slots;  // NULL: no cache
    Cache cache;
    const RopePair* pairs;
    float scale;
    float k_over, v_over;  // 1 / k_scale, 1 / v_scale
    int32_t tokens, heads, kv_heads, n_pairs;
    int32_t x_dtype, y_dtype, cache_dtype;
    int32_t adjacent, inverse;
    FastDiv per_token, per_head, by_pairs;  // items of a token and of a head; n_pairs
};
hipError_t launch_rope(const RopeArgs& a, int head_dim, hipStream_t s);

// ---- attn_append_i8.hip --------------------------------------------------------------
constexpr int kMaxI8Dim = 256;  // head_dim

struct AppendI8Args {
    RopeArgs r;  // per_token: items of q alone
    Scales scales;
    FastDiv by_slices;             // of a q token's items
    uint32_t kv_wgs, q_groups;     // workgroups for k and v, in front; groups of q tokens
    uint32_t chunk, wg_heads;      // tokens whose runs a workgroup takes, of wg_heads heads
    FastDiv by_head_groups;
};
hipError_t launch_append_i8(AppendI8Args& a, int head_dim, hipStream_t s);

// ---- attn_read.hip -------------------------------------------------------------------
struct ReadArgs {
    Cache cache;
    Scales scales;
    const int32_t *tables, *starts, *first;
    int64_t table_stride;
    uint32_t requests, max_len;
    int64_t tokens;
    uint8_t *k_out, *v_out;
    int64_t k_stride, v_stride;  // bytes
    int32_t kv_heads, out_dtype, cache_dtype;
    FastDiv per_head, per_token;  // items of a head, and of a token
};
hipError_t launch_read(const ReadArgs& a, hipStream_t s);

// ---- attn_decode_*.hip ---------------------------------------------------------------
// Whether a call reads keys and values past the caches (loads marked as not used again),
// with `keys` of each key head at most: where these are 128 MiB or more, which the caches (256
// MB, and a step's weights between two calls) would not hold for the next, and where lines of
// 128 bytes are not shared by heads, whose waves read them each at its own time.  Nor where
// several rows, or tiles of heads, read the same keys.  Measured, with and without (us): one
// row of 131071 keys, 8 heads of 128, bf16 90.3 / 98.4; 128 rows of up to 12000, e4m3 245 /
// 271; 16 of up to 4000 (196 MB) 40.4 / 42.6, of 2000 27.7 / 27.4; of heads of 64 in e4m3,
// token after token of a head 71.8 / 75.5, head after head (64 bytes each) 95.8 / 84.8;
// 32 heads of one key head 33.2 / 24.8.
inline bool decode_streams(const Cache& c, int kv_heads, int head_dim, bool f8, int64_t keys) {
    const int row_bytes = head_dim * (f8 ? 1 : 2);
    const bool whole_lines = row_bytes % 128 == 0 ? c.token_stride % 128 == 0 : head_dim % 64 == 0 && c.token_stride == row_bytes;
    const bool aligned = (((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.head_stride | (uintptr_t)c.page_stride) & 127) == 0;
    const int64_t most = keys < (int64_t)c.slots ? keys : (int64_t)c.slots;
    return whole_lines && aligned && 2 * most * kv_heads * row_bytes >= 128 << 20;
}

// A row of several parts (parts > 1), in shares first_share on.
struct Split {
    uint32_t row, first_share, parts;
};

struct DecodeArgs {
    Cache cache;
    const uint8_t* q;
    uint8_t* out;
    float* lse;
    const int32_t *lens, *rows, *tables;
    int64_t q_stride, out_stride;  // bytes
    int64_t table_stride;
    uint32_t n_rows, requests, max_len;  // max_len = max_pages * page_size
    uint32_t window;                     // keys that a row sees at most
    int32_t q_heads, kv_heads, group, head_tiles;
    int32_t out_f32;
    int32_t wide;  // a key's place in the cache takes more than 32 bits
    float scale;  // of a raw product, in powers of two: scale * k_scale * log2(e)
    // Shares of the call's tiles for each of the units = kv_heads * head_tiles, at most, and
    // those that waves are launched for.
    uint32_t shares, launch_shares;
    FastDiv by_units, by_head_tiles;
    // What the join reads: entries of split rows, and for each row (by_row: there are at
    // most as many as shares) or each share the row that is split there.
    float* part_acc;  // [shares][2][q_heads][head_dim]
    float2* part_ml;  // [shares][2][q_heads]: maximum, sum
    Split* split;     // [shares]
    int32_t by_row;
    int32_t uncut;   // shares are rows, whatever their lengths, and there is no join
    int32_t whole;   // a row of a unit to a workgroup, and no join
    int32_t stream;  // keys and values are read past the caches
};

struct DecodeI8Args : DecodeArgs {
    Scales scales;
};

// log(sum of exponentials) from a base in powers of two and the sum above it, whose exponent
// joins the base first (fp16's sums are 2^15 up: the two nearly cancel).
__device__ __forceinline__ float log_sum(float m, float l) {
    const float e = (float)(__builtin_amdgcn_frexp_expf(l) - 1);
    return l == 0 ? -INFINITY : (m + e + __builtin_amdgcn_logf(2.0f * __builtin_amdgcn_frexp_mantf(l))) * 0.693147180559945309f;
}

// Shares of a call, at most.
uint32_t decode_shares(int kv_heads, int head_tiles);

// The parts of split rows joined into out and lse; after launch_decode_*.
hipError_t launch_join(const DecodeArgs& a, int head_dim, int out_dtype, hipStream_t s);

hipError_t launch_decode_bf16(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s);
hipError_t launch_decode_f16(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s);
hipError_t launch_decode_i8_bf16(const DecodeI8Args& a, int head_dim, hipStream_t s);
hipError_t launch_decode_i8_f16(const DecodeI8Args& a, int head_dim, hipStream_t s);

// ---- attn_prompt_*.hip ---------------------------------------------------------------
struct PromptArgs {
    Cache cache;
    Scales scales;
    const uint8_t* q;
    uint8_t* out;
    float* lse;
    const int32_t *lens, *starts, *tables;
    int64_t q_stride, out_stride;  // bytes
    int64_t table_stride;
    uint32_t rows, requests, max_len, window;
    int32_t q_heads, group;
    FastDiv by_tokens, by_heads;      // query tokens and heads of a tile
    FastDiv by_units, by_head_tiles;  // units: key heads times tiles of their query heads
    int32_t negative;  // the scale's sign
    float scale;       // its magnitude, times k_scale and log2(e)
    int32_t waves;     // of a workgroup, 32 rows each
    uint32_t tiles;    // of query tokens, at most
    uint32_t splits;   // workgroups that share a tile's keys
    float* part_acc;   // [tiles * units][splits][tile rows][head_dim]
    float2* part_ml;   // [tiles * units][splits][tile rows]
};
hipError_t launch_prompt_bf16(const PromptArgs& a, int head_dim, int cache_dtype, bool out_f32, hipStream_t s);
hipError_t launch_prompt_f16(const PromptArgs& a, int head_dim, int cache_dtype, bool out_f32, hipStream_t s);
hipError_t launch_prompt_join(const PromptArgs& a, int head_dim, int out_dtype, hipStream_t s);

}  // namespace attn
