// Attention of runs of query tokens over a paged cache (openmini_attn_prompt).
//
// A tile is some query tokens of one request times the query heads of one key head: 32 rows to
// a wave.  For each step of 64 keys (32 in heads of 192 and 256), which the workgroup brings
// into LDS for all its waves as 16-bit elements, a wave computes
//   S^T = K q^T, p = 2^(s - m), O^T += V^T P^T
// on 32 x 32 x 16 tiles with its rows as the columns, m and l the running maximum and sum of
// each.  The C layout of S^T gives lane (h = lane / 32, column lane % 32) rows 8 a + 4 h + b,
// the B layout of P^T wants k = 8 h .. 8 h + 7 of the column in the same lane.  With keys put
// into K's rows with bits 2 and 3 of their number exchanged, the two are the same keys: the
// probabilities go from one product to the next without leaving their lane, a group of eight
// neighbours to each operand, which share a block and its scale.
//
// V lies in LDS transposed, [dimension][key]: a thread brings four keys of four dimensions and
// transposes them by byte permutations on the way.
//
// 8-bit integers are exact in 16 bits; their blocks' scales act on 32-bit numbers: a key's on
// the score, a value's as its logarithm in the exponent, so that p v_scale against the row's base is what
// is rounded to 16 bits (at most 2^15 in fp16 and 2^8 in bf16 parts, whatever the scales) and l adds p
// v_scale / v_scale.  The logarithm and its sum are off by up to 2^-20 for scales near 2^-5 (measured: 2^-21
// of sum p |v|), 2^-17 near 2^-60.
//
// The loads of a step are issued more than a step ahead of their use and its page three (heads of 192 and 256: a
// step and two, with another workgroup on the CU); two buffers, one barrier a step.  What comes goes to LDS beside the matrix instructions of the first product.
// Accumulators are scaled only where a maximum has passed its base by 2^8 (bf16 parts), 2^4 (one fp16
// part) or at all (two fp16 parts and what they leave): with 32 rows to a wave one of them grows in most steps.
//
// Bound by the issue of instructions: a step of 64 keys takes a wave 2 us, alone on its SIMD or with
// another, of which the matrix unit is busy for .4 (heads of 128); matrix and vector instructions of
// the two waves run at the same time for two fifths of that only.  Measured (MI355X, us, calls in a row once
// clocks have settled; the first twenty on an idle card take up to a third more): 8191 tokens of 64 / 8 heads of
// 128 1165 to 1240, 885 to 945 TFLOP/s (a large product of the library 1350); 4096 tokens of 32 / 8 heads of 64, 96,
// 128, 192, 256 142, 159, 162, 283, 364, of 128 on a bf16, fp16, e4m3 cache 169, 176, 168 (so conversions are not what
// binds), with fp32 out on 8-bit integers, bf16, fp16 254, 267, 248; 211 tokens of 64 / 8 heads of 128 13.6; 815 tokens
// in six pieces behind up to 1659 keys, 32 / 8 heads of 64 in fp16, fp32 out, 38.
// What gave nothing or less: a second product a step later, for
// half of the waves or among the exponentials (1.24, 1.47 ms of 1.26), wave priorities, 128 keys
// a step, three waves a SIMD of 32 keys a step (1.31 of 1.18), rows out through LDS.
#pragma once

#include "attn_decode.hpp"
#include "attn_runs.hpp"

namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(BF16, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(F16, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Over the two lanes of a column.
__device__ __forceinline__ float halves_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Elements without a finite value among the two of u.
template <class T>
__device__ __forceinline__ uint32_t not_finite(uint32_t u) {
    constexpr uint32_t kAll = std::is_same_v<T, BF16> ? 0x7F80u : 0x7C00u;
    return ((u & kAll) == kAll ? 0xFFFFu : 0u) | ((u >> 16 & kAll) == kAll ? 0xFFFF0000u : 0u);
}

// A tile's place: slot t of the call's tiles; of n tokens each, run r has those from
// (starts[r] + r (n - 1)) / n on, at least as many as it needs.
struct PromptTile {
    uint32_t run, token0, tokens;  // tokens: 0 for a slot that no run needs
    uint32_t kv, head0, heads;     // its key head, its first query head, its heads
};
__device__ __forceinline__ PromptTile prompt_tile(const int32_t* starts, uint32_t rows, uint32_t requests, FastDiv by_tokens, uint32_t slot,
                                                  uint32_t unit, FastDiv by_head_tiles, FastDiv by_heads, int32_t group) {
    auto start = [&](uint32_t r) { return min((uint32_t)max(starts[r], 0), rows); };
    PromptTile t;
    t.tokens = 0;
    t.run = find_run(requests, slot, [&](uint32_t r) { return by_tokens.div(start(r) + r * (by_tokens.d - 1)); });
    t.kv = by_head_tiles.div(unit);
    const uint32_t part = (unit - t.kv * by_head_tiles.d) * by_heads.d;
    t.head0 = t.kv * (uint32_t)group + part;
    t.heads = min(by_heads.d, (uint32_t)group - part);
    t.token0 = 0;
    if (t.run >= requests) return t;
    const uint32_t first = start(t.run), end = start(t.run + 1);
    const uint64_t at = first + (uint64_t)(slot - by_tokens.div(first + t.run * (by_tokens.d - 1))) * by_tokens.d;
    if (at >= end) return t;
    t.token0 = (uint32_t)at;
    t.tokens = min(by_tokens.d, end - t.token0);
    return t;
}

// kPer: waves a SIMD.
template <int D, class T, Elem E, bool kF32, int W, int kPer>
__global__ __launch_bounds__(64 * W, kPer) void prompt_kernel(PromptArgs a) {
    // of the second product: byte caches fit both types, fp16 has the finer step and bf16 the
    // range that exact parts need.  16-bit outputs take one part of a probability, off by as much as their
    // own rounding: rms against 64 bits, relative, with one part and with all, fp16 on 8-bit integers 2.4e-4 /
    // 2.1e-4, on fp16 2.5e-4 / 2.0e-4, bf16 on 8-bit integers 1.7e-3 / 1.7e-3, on bf16 2.0e-3 / 1.6e-3; 4096
    // tokens of 32 heads 162 / 254 us
    using P = std::conditional_t<E == kHalf, T, std::conditional_t<kF32, BF16, F16>>;
    constexpr int kParts = kF32 ? P::kExactParts : 1;
    constexpr bool kLow = kF32 && P::kNarrow;  // as in decode attention: what two fp16 parts leave
    constexpr int kThreads = 64 * W, kKeys = prompt_keys(D), kSub = kKeys / 32;
    constexpr int kEl = E == kHalf ? 2 : 1;
    constexpr int kSteps = D / 16, kTiles = D / 32;
    // bytes of a row in LDS: 16 more than its elements, so that the eight lanes of an access, each at
    // its row, fall on different banks, and all of a lane's reads are at fixed distances
    constexpr int kKRow = D * 2 + 16, kVRow = kKeys * 2 + 16;
    constexpr int kKLoads = (8 * D * kEl / 16 + 63) / 64, kVLoads = (D / 2 + 63) / 64;
    constexpr int kGroups = kKeys / 8;
    constexpr int kOwn = kGroups / W;  // groups that a wave brings
    constexpr int kSets = D <= 128 || kPer == 1 ? 2 : 1;  // steps whose data are on their way
    static_assert(kGroups % W == 0);

    constexpr int kKBytes = kKeys * kKRow, kVBytes = D * kVRow;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kKBytes + 2 * kVBytes];  // both arrays, of two steps
    // of eight keys: their score's factor, the logarithm and the reciprocal of their values' scale,
    // and whether their page is in the cache
    __shared__ __attribute__((aligned(16))) f32x4 group_lds[2][kGroups];
    __shared__ uint32_t flags[3];  // of a step: 1 keys on no page, 2 values without a number where rows differ
    __shared__ int32_t bounds[4][W];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    const uint32_t back = a.by_units.div(blockIdx.x), unit = blockIdx.x - back * a.by_units.d, slot = a.tiles - 1 - back;
    const PromptTile tile = prompt_tile(a.starts, a.rows, a.requests, a.by_tokens, slot, unit, a.by_head_tiles, a.by_heads, a.group);
    if (!tile.tokens) return;

    // the lane's row; rows past the tile's repeat its last
    const uint32_t at_row = (uint32_t)(wave * kWaveRows + col), at_token = a.by_heads.div(at_row), at_head = at_row - at_token * a.by_heads.d;
    const bool real = at_token < tile.tokens && at_head < tile.heads;
    const uint32_t row = tile.token0 + min(at_token, tile.tokens - 1), head = tile.head0 + min(at_head, tile.heads - 1);
    const bool any_real = __any(real);  // a wave without a row of its own sees nothing
    const int32_t hi = any_real ? min(max(a.lens[row], 0), (int32_t)a.max_len) : 0, lo = (int32_t)max((uint32_t)hi, a.window) - (int32_t)a.window;

    u32x4 qf[kSteps];
    {
        const uint8_t* q = a.q + row * a.q_stride + (int64_t)head * D * 2 + half * 16;
        const uint32_t flip = a.negative ? 0x80008000u : 0;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) qf[st] = *reinterpret_cast<const u32x4*>(q + st * 32) ^ flip;
    }

    // the keys that the wave's rows see, all and some of them; the workgroup's
    int32_t hi_most = hi, hi_least = hi, lo_most = lo, lo_least = hi ? lo : INT32_MAX;
#pragma unroll
    for (int by = 1; by < 32; by *= 2) {
        hi_most = max(hi_most, __shfl_xor(hi_most, by));
        hi_least = min(hi_least, __shfl_xor(hi_least, by));
        lo_most = max(lo_most, __shfl_xor(lo_most, by));
        lo_least = min(lo_least, __shfl_xor(lo_least, by));
    }
    hi_most = __builtin_amdgcn_readfirstlane(hi_most);
    hi_least = __builtin_amdgcn_readfirstlane(hi_least);
    lo_most = __builtin_amdgcn_readfirstlane(lo_most);
    lo_least = __builtin_amdgcn_readfirstlane(lo_least);
    if (lane == 0) {
        bounds[0][wave] = hi_most;
        bounds[1][wave] = any_real ? hi_least : INT32_MAX;
        bounds[2][wave] = lo_most;
        bounds[3][wave] = lo_least;
    }
    if (tid < 3) flags[tid] = 0;
    __syncthreads();
    int32_t all_hi = bounds[0][0], each_hi = bounds[1][0], each_lo = bounds[2][0], all_lo = bounds[3][0];  // wave 0 has rows
#pragma unroll
    for (int w = 1; w < W; ++w) {
        all_hi = max(all_hi, bounds[0][w]);
        each_hi = min(each_hi, bounds[1][w]);
        each_lo = max(each_lo, bounds[2][w]);
        all_lo = min(all_lo, bounds[3][w]);
    }
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    each_hi = __builtin_amdgcn_readfirstlane(each_hi);
    each_lo = __builtin_amdgcn_readfirstlane(each_lo);
    all_lo = __builtin_amdgcn_readfirstlane(min(all_lo, all_hi));
    // steps [from, to) of the tile's keys: the split's share of them
    uint32_t from = (uint32_t)all_lo / kKeys, to = ((uint32_t)all_hi + kKeys - 1) / kKeys;
    if (a.splits > 1) {
        const uint32_t each = (to - from + a.splits - 1) / a.splits;
        from = min(from + blockIdx.y * each, to);
        to = min(from + each, to);
    }

    auto k_lds = [&](int buf) { return lds + buf * kKBytes; };
    auto v_lds = [&](int buf) { return lds + 2 * kKBytes + buf * kVBytes; };
    const int32_t* table = a.tables + tile.run * a.table_stride;
    const uint8_t* k_base = a.cache.k + tile.kv * a.cache.head_stride;
    const uint8_t* v_base = a.cache.v + tile.kv * a.cache.head_stride;
    const int32_t last = all_hi - 1;

    // What a wave brings of a step: groups of eight keys, which share a page and a block, so that their
    // place is worked out once, in scalar registers; a lane pieces of 16 bytes of a key, and units of 4 keys
    // and 4 dimensions of the values.
    constexpr int kRowPieces = D * kEl / 16;
    auto piece_of = [&](int i) __attribute__((always_inline)) { return lane + 64 * i; };
    // Bytes: a piece is two accesses of LDS, of which eight lanes take four pieces of two keys, whose
    // rows lie an odd number of accesses apart.
    constexpr bool kPairs = kEl == 1 && kRowPieces % 4 == 0;
    auto key_of = [&](int i) __attribute__((always_inline)) { return kPairs ? piece_of(i) / (2 * kRowPieces) * 2 + (piece_of(i) >> 2 & 1) : piece_of(i) / kRowPieces; };
    auto part_of = [&](int i) __attribute__((always_inline)) {
        return kPairs ? (piece_of(i) >> 3) % (kRowPieces / 4) * 4 + (piece_of(i) & 3) : piece_of(i) % kRowPieces;
    };
    auto has_piece = [&](int i) __attribute__((always_inline)) { return (8 * kRowPieces) % 64 == 0 || piece_of(i) < 8 * kRowPieces; };
    auto has_unit = [&](int i) __attribute__((always_inline)) { return (D / 2) % 64 == 0 || piece_of(i) < D / 2; };
    int64_t k_off[kKLoads], v_off[kVLoads];
#pragma unroll
    for (int i = 0; i < kKLoads; ++i)
        k_off[i] = key_of(i) * a.cache.token_stride + part_of(i) * 16;
#pragma unroll
    for (int i = 0; i < kVLoads; ++i)
        v_off[i] = piece_of(i) / (D / 4) * 4 * a.cache.token_stride + piece_of(i) % (D / 4) * 4 * kEl;
    struct Pages {
        int32_t page[kOwn];  // the same in all lanes, not yet in a scalar register
        uint32_t in_page[kOwn];
    };
    auto pages_of = [&](uint32_t step) __attribute__((always_inline)) {
        Pages p;
#pragma unroll
        for (int g = 0; g < kOwn; ++g) {
            const uint32_t key = min(step * kKeys + 8 * (uint32_t)(kOwn * wave + g), (uint32_t)last & ~7u);
            const uint32_t at = a.cache.page.div(key);
            uint32_t v_at = at;
            asm("" : "+v"(v_at));  // a vector load: a scalar one would be waited for with the reads of LDS
            p.page[g] = table[v_at];
            p.in_page[g] = key - at * a.cache.page.d;
        }
        return p;
    };
    auto in_cache = [&](int32_t page) __attribute__((always_inline)) { return (uint32_t)page < a.cache.n_pages; };
    struct Raw {
        u32x4 k[kKLoads];
        uint32_t v[kVLoads][4][kEl];
        float k_scale, v_scale;
        bool paged;
    };
    auto load_group = [&](int32_t page, uint32_t in_page, Raw& r) __attribute__((always_inline)) {
        page = __builtin_amdgcn_readfirstlane(page);
        r.paged = in_cache(page);
        const int64_t place = (r.paged ? page * a.cache.page_stride : 0) + (int64_t)in_page * a.cache.token_stride;
#pragma unroll
        for (int i = 0; i < kKLoads; ++i)
            if (has_piece(i)) r.k[i] = *reinterpret_cast<const u32x4*>(k_base + place + k_off[i]);
#pragma unroll
        for (int i = 0; i < kVLoads; ++i)
            if (has_unit(i)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) attn::load<4 * kEl, false>(v_base + (place + j * a.cache.token_stride) + v_off[i], r.v[i][j]);
            }
        if constexpr (E == kI8) {
            int64_t at = (r.paged ? page : 0) * a.scales.page_stride + (int64_t)(in_page >> a.scales.shift) * a.scales.block_stride +
                         tile.kv * a.scales.head_stride;
            asm("" : "+v"(at));
            r.k_scale = a.scales.k[at];
            r.v_scale = a.scales.v[at];
        }
    };
    auto load = [&](const Pages& p, Raw* r) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < kOwn; ++g) load_group(p.page[g], p.in_page[g], r[g]);
    };
    auto store_group = [&](Raw& r, int group, uint32_t step, int buf, int flag) __attribute__((always_inline)) {
        const int32_t key0 = (int32_t)(step * kKeys);
        const bool partial = key0 < each_lo || key0 + kKeys > each_hi;
#pragma unroll
        for (int i = 0; i < kKLoads; ++i)
            if (has_piece(i)) {
                const int key = 8 * group + key_of(i);
                const int r_lds = (key & ~12) | (key & 4) << 1 | (key & 8) >> 1;
                u32x4* to = reinterpret_cast<u32x4*>(k_lds(buf) + r_lds * kKRow + part_of(i) * (32 / kEl));
                if constexpr (E == kHalf) {
                    *to = r.k[i];
                } else {
                    const u32x4 w = r.k[i];
                    to[0] = u32x4{from_byte<T, E, false>(w[0]), from_byte<T, E, true>(w[0]), from_byte<T, E, false>(w[1]), from_byte<T, E, true>(w[1])};
                    to[1] = u32x4{from_byte<T, E, false>(w[2]), from_byte<T, E, true>(w[2]), from_byte<T, E, false>(w[3]), from_byte<T, E, true>(w[3])};
                }
            }
#pragma unroll
        for (int i = 0; i < kVLoads; ++i)
            if (has_unit(i)) {
                const int kg = 2 * group + piece_of(i) / (D / 4), quad = piece_of(i) % (D / 4);
                u32x2 v[4];  // of each dimension, four keys
                if constexpr (E == kHalf) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                        v[e] = u32x2{__builtin_amdgcn_perm(r.v[i][1][e / 2], r.v[i][0][e / 2], sel),
                                     __builtin_amdgcn_perm(r.v[i][3][e / 2], r.v[i][2][e / 2], sel)};
                    }
                } else {
                    const uint32_t l01 = __builtin_amdgcn_perm(r.v[i][1][0], r.v[i][0][0], 0x05010400u);
                    const uint32_t h01 = __builtin_amdgcn_perm(r.v[i][1][0], r.v[i][0][0], 0x07030602u);
                    const uint32_t l23 = __builtin_amdgcn_perm(r.v[i][3][0], r.v[i][2][0], 0x05010400u);
                    const uint32_t h23 = __builtin_amdgcn_perm(r.v[i][3][0], r.v[i][2][0], 0x07030602u);
                    v[0] = u32x2{from_byte<P, E, false>(l01), from_byte<P, E, false>(l23)};
                    v[1] = u32x2{from_byte<P, E, true>(l01), from_byte<P, E, true>(l23)};
                    v[2] = u32x2{from_byte<P, E, false>(h01), from_byte<P, E, false>(h23)};
                    v[3] = u32x2{from_byte<P, E, true>(h01), from_byte<P, E, true>(h23)};
                }
                if constexpr (E != kI8)  // 0 * NaN is NaN: nothing past the rows' keys, and who sees what is left is told
                    if (partial || !r.paged) {
                        const int32_t key = r.paged ? key0 + 4 * kg : INT32_MAX - 3;
                        const u32x2 keep = {(key <= last ? 0xFFFFu : 0) | (key + 1 <= last ? 0xFFFF0000u : 0),
                                            (key + 2 <= last ? 0xFFFFu : 0) | (key + 3 <= last ? 0xFFFF0000u : 0)};
                        uint32_t bad = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[e] &= keep;
                            bad |= not_finite<P>(v[e][0]) | not_finite<P>(v[e][1]);
                        }
                        if (bad) atomicOr(&flags[flag], 2u);
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) *reinterpret_cast<u32x2*>(v_lds(buf) + (quad + D / 4 * e) * kVRow + kg * 8) = v[e];
            }
        if (lane == 0) {
            f32x4 g = {a.scale, 0, 1, r.paged ? 1.0f : 0.0f};
            if constexpr (E == kI8) {
                const float v = r.v_scale, k = __builtin_fmaf(a.scale, r.k_scale, r.k_scale - r.k_scale);  // of infinity NaN, as in decode attention
                g[0] = k < 1e-37f ? 1e-37f : k;  // -inf times 0 is NaN
                const float up = v < 8.673617379884035e-19f ? 8.673617379884035e-19f : v;  // 2^-60
                g[1] = fabsf(v) <= 0x1p126f ? __builtin_amdgcn_logf(up) : __uint_as_float(0x7FC00000u);  // past it the reciprocal is 0
                g[2] = __builtin_amdgcn_rcpf(up);  // within 2^-23
            }
            group_lds[buf][group] = g;
            if (!r.paged && key0 + 8 * group <= last) atomicOr(&flags[flag], 1u);
        }
    };

    auto store = [&](Raw* r, uint32_t step, int buf, int flag) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < kOwn; ++g) store_group(r[g], kOwn * wave + g, step, buf, flag);
    };

    f32x16 acc[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0;
    float m = -INFINITY, l = 0;

    // Dimension 4 q + e is row q + D / 4 e of V: the lanes that write side by side are at neighbouring
    // rows, and a lane's accumulators hold 16 neighbouring dimensions: row 32 t + 8 a + 4 half + b
    // of tile t is accumulator 4 a + b.
    auto v_at = [&](int buf, int row, int slot) __attribute__((always_inline)) { return v_lds(buf) + row * kVRow + slot * 16; };
    // Values without a number in a step that not every row sees whole: their dimension is NaN for
    // the rows that see them, and they are taken out for the others.  Rare, and slow.
    auto part_ways = [&](uint32_t step, int buf) __attribute__((always_inline)) {
        const int32_t key0 = (int32_t)(step * kKeys);
        for (int key = 0; key < kKeys; ++key) {
            const bool seen = key0 + key >= lo && key0 + key < hi && group_lds[buf][key / 8][3] != 0;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int row = 32 * t + 8 * (i >> 2) + 4 * half + (i & 3);
                    const uint32_t v = *reinterpret_cast<const uint16_t*>(v_at(buf, row, key / 8) + key % 8 * 2);
                    if (seen && not_finite<P>(v)) acc[t][i] = __uint_as_float(0x7FC00000u);
                }
        }
        __syncthreads();
        for (int i = tid; i < D * kVRow / 4; i += kThreads) {
            uint32_t* v = reinterpret_cast<uint32_t*>(v_lds(buf)) + i;
            *v &= ~not_finite<P>(*v);
        }
        __syncthreads();
    };

    // The accumulators are scaled only where a maximum passes its base by more than 2^kLag: p
    // reaches as much then.  fp16's is 2^(15 - kLag) at the base, so 2^15 at most, below the largest
    // number; parts that leave out what lies low have no room for it.
    constexpr float kLag = !P::kNarrow ? 8 : kLow ? 0 : 4;
    auto base_of = [](float top) { return P::kNarrow && fabsf(top) < 8388608.0f ? top - (15 - kLag) : top; };
    f32x16 sc[kSub];  // scores of a step, then its probabilities
    bool low = false;
    // Whether the wave's rows see any of the step.
    auto sees = [&](uint32_t step) __attribute__((always_inline)) {
        const int32_t key0 = (int32_t)(step * kKeys);
        return key0 < hi_most && key0 + kKeys > lo_least;
    };
    auto scores = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[u][i] = 0;
        const uint8_t* k_row = k_lds(buf) + col * kKRow + half * 16;
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
#pragma unroll
            for (int u = 0; u < kSub; ++u)
                sc[u] = mfma32(T{}, *reinterpret_cast<const u32x4*>(k_row + 32 * u * kKRow + st * 32), qf[st], sc[u]);
    };
    // The scores become probabilities; m and l.
    auto probabilities = [&](uint32_t step, int buf, uint32_t said) __attribute__((always_inline)) {
        const int32_t key0 = (int32_t)(step * kKeys);
        f32x4 group[2 * kSub];
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) group[j] = E == kI8 ? group_lds[buf][2 * j + half] : f32x4{a.scale, 0, 1, 1};
        float least = INFINITY;  // before the mask: an edge is not low
        if constexpr (kLow)
#pragma unroll
            for (int j = 0; j < 2 * kSub; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) least = fminf(least, sc[j / 2][8 * (j & 1) + i]);
        if (key0 < lo_most || key0 + kKeys > hi_least || (said & 1)) {
#pragma unroll
            for (int j = 0; j < 2 * kSub; ++j) {
                const uint32_t from_lo = (uint32_t)(key0 + 16 * j + 8 * half - lo);
                const uint32_t span = group_lds[buf][2 * j + half][3] != 0 ? (uint32_t)(hi - lo) : 0;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sc[j / 2][8 * (j & 1) + i] = from_lo + i < span ? sc[j / 2][8 * (j & 1) + i] : -INFINITY;
                // nor are the scales of a group that the row does not see
                if constexpr (E == kI8) {
                    const bool some = from_lo + 7 < span + 7 && span != 0;
                    group[j] = f32x4{some ? group[j][0] : 1, some ? group[j][1] : 0, some ? group[j][2] : 0, 0};
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
            float t = sc[j / 2][8 * (j & 1)];
#pragma unroll
            for (int i = 1; i < 8; ++i) t = fmaxf(t, sc[j / 2][8 * (j & 1) + i]);
            top = fmaxf(top, E == kI8 ? __builtin_fmaf(t, group[j][0], group[j][1]) : t);
        }
        if constexpr (E != kI8) top *= a.scale;
        const float lift = base_of(halves_max(top));
        if (__any(lift > m + kLag)) {
            const float up = fmaxf(m, lift), by = exp2_of(m - above(up));
            m = up;
            l *= by;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) acc[t] *= by;
        }
        const float base = above(m);
        if constexpr (kLow) low = __any(least * a.scale < base - 2.0f);
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
            const float off = E == kI8 ? group[j][1] - base : -base, by = E == kI8 ? group[j][0] : a.scale;
            float sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = exp2_of(__builtin_fmaf(sc[j / 2][8 * (j & 1) + i], by, off));
                sc[j / 2][8 * (j & 1) + i] = s;
                sum += s;
            }
            l = E == kI8 ? __builtin_fmaf(sum, group[j][2], l) : l + sum;
        }
    };
    constexpr float kUp = 549755813888.0f;  // 2^39
    auto product = [&](int buf) __attribute__((always_inline)) {
        // p of groups 2 j and 2 j + 1 in parts, which leave their rest in it
        auto parts = [&](int j, float* p, auto add_tag) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                u32x4 pf;
                float minus = -1;
                if constexpr (P::kNarrow) asm("" : "+s"(minus));  // else a conversion and a subtraction
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    pf[i / 2] = P::pair(p[i], p[i + 1]);
                    if constexpr (P::kNarrow) {  // from the pair, one instruction each: not rounded a second time
                        asm("" : "+v"(pf[i / 2]));
                        p[i] = __builtin_fmaf(P::low(pf[i / 2]), minus, p[i]);
                        p[i + 1] = __builtin_fmaf(P::high(pf[i / 2]), minus, p[i + 1]);
                    } else {
                        p[i] -= P::low(pf[i / 2]);
                        p[i + 1] -= P::high(pf[i / 2]);
                    }
                }
                if constexpr (decltype(add_tag)::value)
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        acc[t] = mfma32(P{}, *reinterpret_cast<const u32x4*>(v_at(buf, 32 * t + col, 2 * j + half)), pf, acc[t]);
            }
        };
        auto p_of = [&](int j, float* p) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = sc[j / 2][8 * (j & 1) + i];
        };
        float p[8];
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
            p_of(j, p);
            parts(j, p, std::true_type{});
        }
        if constexpr (kLow) {
            if (!low) return;
            // not the reads and parts above, kept in more registers than there are
            asm volatile("" ::: "memory");
#pragma unroll
            for (int u = 0; u < kSub; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(sc[u][i]));
            // what two parts leave of p < 2^-2, 2^39 up
#pragma unroll
            for (int t = 0; t < kTiles; ++t) acc[t] *= kUp;
#pragma unroll
            for (int j = 0; j < 2 * kSub; ++j) {
                p_of(j, p);
                parts(j, p, std::false_type{});
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = sc[j / 2][8 * (j & 1) + i] < 0.25f ? p[i] * kUp : 0.0f;
                parts(j, p, std::true_type{});
            }
#pragma unroll
            for (int t = 0; t < kTiles; ++t) acc[t] *= 1.0f / kUp;
        }
    };

    if (from < to) {
        Raw raw[kSets][kOwn];  // of steps from + 0, 2, ... and from + 1, 3, ...
        const uint32_t end = to - 1;
        Pages then;
        {
            const Pages first = pages_of(from), second = pages_of(min(from + 1, end));
            then = kSets == 2 ? pages_of(min(from + 2, end)) : second;
            load(first, raw[0]);
            if constexpr (kSets == 2) load(second, raw[1]);
        }
        store(raw[0], from, 0, 0);
        __syncthreads();
        int flag = 0;
        // Past the last step it is loaded and stored again: no branches around loads, whose waits would
        // be for all.
        auto one_step = [&](uint32_t step, auto buf_tag) __attribute__((always_inline)) {
            constexpr int buf = decltype(buf_tag)::value;
            const int next_flag = flag == 2 ? 0 : flag + 1;
            // the page before the loads: a wait for it is none for them
            const Pages later = pages_of(min(step + 1 + kSets, end));
            load(then, raw[kSets == 2 ? buf : 0]);
            then = later;
            const uint32_t said = flags[flag];
            if constexpr (E != kI8)
                if (said & 2) part_ways(step, buf);
            if constexpr (kSets == 2) {
                if (sees(step)) {
                    scores(buf);
                    store(raw[buf ^ 1], min(step + 1, end), buf ^ 1, next_flag);  // beside the matrix instructions
                    probabilities(step, buf, said);
                    product(buf);
                } else {
                    store(raw[buf ^ 1], min(step + 1, end), buf ^ 1, next_flag);
                }
            } else {
                if (sees(step)) {
                    scores(buf);
                    probabilities(step, buf, said);
                    product(buf);
                }
                store(raw[0], min(step + 1, end), buf ^ 1, next_flag);
            }
            // the flags of the step after the next: read last a step ago, before a barrier
            if (tid == 0) flags[next_flag == 2 ? 0 : next_flag + 1] = 0;
            flag = next_flag;
            __syncthreads();
        };
        for (uint32_t step = from;; step += 2) {
            one_step(step, std::integral_constant<int, 0>{});
            if (step == end) break;
            one_step(step + 1, std::integral_constant<int, 1>{});
            if (step + 1 == end) break;
        }
    }

    l = halves_sum(l);
    if (!real) return;
    // the lane's accumulators, four neighbouring dimensions at a time
    auto each_four = [&](auto&& f) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[(2 * k + D / 16 * e) / 8][(2 * k + D / 16 * e) % 8 / 2 * 4 + b];
                f(32 * k + 16 * half + 4 * b, v);
            }
    };
    if (a.splits > 1) {
        const int64_t entry = (((int64_t)slot * a.by_units.d + unit) * a.splits + blockIdx.y) * (W * kWaveRows) + at_row;
        float* o = a.part_acc + entry * D;
        each_four([&](int dim, f32x4 v) { *reinterpret_cast<f32x4*>(o + dim) = v; });
        if (half == 0) a.part_ml[entry] = make_float2(m, l);
        return;
    }
    const float over = l > 0 || l != l ? a.cache.v_scale / l : 0.0f;
    uint8_t* out = a.out + row * a.out_stride + (int64_t)head * D * (kF32 ? 4 : 2);
    each_four([&](int dim, f32x4 v) {
        v *= over;
        if constexpr (kF32)
            *reinterpret_cast<f32x4*>(out + dim * 4) = v;
        else
            *reinterpret_cast<u32x2*>(out + dim * 2) = u32x2{T::pair(v[0], v[1]), T::pair(v[2], v[3])};
    });
    if (a.lse && half == 0) a.lse[(int64_t)row * a.q_heads + head] = log_sum(m, l);
}

template <int D, class T, Elem E, bool kF32, int W>
hipError_t launch_prompt_out(const PromptArgs& a, hipStream_t s) {
    const dim3 grid(a.tiles * a.by_units.d, a.splits), block(64 * W);
    // Two workgroups a CU hide each other's waits, though heads of 192 and 256 have registers for one step's
    // data then, not two, and those of 256 keep 80 to 240 bytes in scratch.  4096 tokens of 32 heads against one
    // workgroup (MI355X, us): of 192 304 / 533 (16-bit caches 313 / 511), of 256 357 / 520 (557 / 572, fp32
    // out 612 / 641).  Heads of 256: 600 tokens (150 workgroups) 49 / 43, 1200 (300) 90 / 80, 2000 (500) 146 / 140, 512 behind 8000 keys
    // (512) 210 / 267, and with what two fp16 parts leave 1100 / 711.
    if constexpr (D == 256)
        if ((E == kHalf && kF32 && T::kNarrow) || (int64_t)grid.x * grid.y <= prompt_alone(D)) {
            hipLaunchKernelGGL((prompt_kernel<D, T, E, kF32, W, 1>), grid, block, 0, s, a);
            return hipGetLastError();
        }
    if constexpr (!(D == 256 && E == kHalf && kF32 && T::kNarrow))
        hipLaunchKernelGGL((prompt_kernel<D, T, E, kF32, W, 2>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <int D, class T, Elem E, int W>
hipError_t launch_prompt_waves(const PromptArgs& a, bool out_f32, hipStream_t s) {
    return out_f32 ? launch_prompt_out<D, T, E, true, W>(a, s) : launch_prompt_out<D, T, E, false, W>(a, s);
}

template <int D, class T, Elem E>
hipError_t launch_prompt_elem(const PromptArgs& a, bool out_f32, hipStream_t s) {
    if constexpr (D <= 128)
        if (a.waves == 8) return launch_prompt_waves<D, T, E, 8>(a, out_f32, s);
    return launch_prompt_waves<D, T, E, 4>(a, out_f32, s);
}

template <int D, class T>
hipError_t launch_prompt_dim(const PromptArgs& a, int cache_dtype, bool out_f32, hipStream_t s) {
    if (cache_dtype == OPENMINI_ATTN_I8) return launch_prompt_elem<D, T, kI8>(a, out_f32, s);
    if (cache_dtype == OPENMINI_ATTN_F8_E4M3) return launch_prompt_elem<D, T, kF8>(a, out_f32, s);
    return launch_prompt_elem<D, T, kHalf>(a, out_f32, s);
}

template <class T>
hipError_t launch_prompt_type(const PromptArgs& a, int head_dim, int cache_dtype, bool out_f32, hipStream_t s) {
    switch (head_dim) {
    case 64: return launch_prompt_dim<64, T>(a, cache_dtype, out_f32, s);
    case 96: return launch_prompt_dim<96, T>(a, cache_dtype, out_f32, s);
    case 128: return launch_prompt_dim<128, T>(a, cache_dtype, out_f32, s);
    case 192: return launch_prompt_dim<192, T>(a, cache_dtype, out_f32, s);
    case 256: return launch_prompt_dim<256, T>(a, cache_dtype, out_f32, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace attn
