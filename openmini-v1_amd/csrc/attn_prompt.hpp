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
// transposes them by byte permutations on the way.  Both arrays are swizzled so that the eight
// lanes of an LDS access fall on different banks.
//
// 8-bit integers are exact in 16 bits; their blocks' scales act on 32-bit numbers: a key's on
// the score, a value's as its logarithm in the exponent, so that p v_scale is what is rounded
// to 16 bits (at most 1, whatever the scales) and l adds p v_scale / v_scale.
//
// The loads of a step are issued a step ahead of their use and its pages two; two buffers,
// one barrier a step.  Bound by the matrix rate for long prompts.
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

// A tile's place: slot t of the call's tiles; run r has those from starts[r] / tokens + r on, at
// least as many as it needs.
struct PromptTile {
    uint32_t run, token0, tokens;  // tokens: 0 for a slot that no run needs
    uint32_t kv, head0, heads;     // its key head, its first query head, its heads
};
__device__ __forceinline__ PromptTile prompt_tile(const int32_t* starts, uint32_t rows, uint32_t requests, FastDiv by_tokens, uint32_t slot,
                                                  uint32_t unit, FastDiv by_head_tiles, FastDiv by_heads, int32_t group) {
    auto start = [&](uint32_t r) { return min((uint32_t)max(starts[r], 0), rows); };
    PromptTile t;
    t.tokens = 0;
    t.run = find_run(requests, slot, [&](uint32_t r) { return by_tokens.div(start(r)) + r; });
    t.kv = by_head_tiles.div(unit);
    const uint32_t part = (unit - t.kv * by_head_tiles.d) * by_heads.d;
    t.head0 = t.kv * (uint32_t)group + part;
    t.heads = min(by_heads.d, (uint32_t)group - part);
    t.token0 = 0;
    if (t.run >= requests) return t;
    const uint32_t first = start(t.run), end = start(t.run + 1);
    const uint64_t at = first + (uint64_t)(slot - by_tokens.div(first) - t.run) * by_tokens.d;
    if (at >= end) return t;
    t.token0 = (uint32_t)at;
    t.tokens = min(by_tokens.d, end - t.token0);
    return t;
}

template <int D, class T, Elem E, bool kF32>
__global__ __launch_bounds__(64 * prompt_waves(D), D <= 128 ? 2 : 1) void prompt_kernel(PromptArgs a) {
    // of the second product: byte caches fit both types, fp16 has the finer step and bf16 the
    // range that exact parts need
    using P = std::conditional_t<E == kHalf, T, std::conditional_t<kF32, BF16, F16>>;
    constexpr int kParts = kF32 ? P::kExactParts : 1;
    constexpr bool kLow = kF32 && P::kNarrow;  // as in decode attention: what two fp16 parts leave
    constexpr int W = prompt_waves(D), kThreads = 64 * W, kKeys = prompt_keys(D), kSub = kKeys / 32;
    constexpr int kEl = E == kHalf ? 2 : 1;
    constexpr int kSteps = D / 16, kTiles = D / 32;
    constexpr int kKRow = (D / 8 + 7) / 8 * 128, kVRow = kKeys * 2;  // bytes of a row in LDS
    constexpr int kKPieces = kKeys * D * kEl / 16, kKLoads = (kKPieces + kThreads - 1) / kThreads;
    constexpr int kVUnits = kKeys / 4 * (D / 4), kVLoads = (kVUnits + kThreads - 1) / kThreads;
    constexpr int kGroups = kKeys / 8;

    __shared__ __attribute__((aligned(16))) uint8_t k_lds[2][kKeys * kKRow], v_lds[2][D * kVRow];
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
    const int32_t hi = min(max(a.lens[row], 0), (int32_t)a.max_len), lo = (int32_t)max((uint32_t)hi, a.window) - (int32_t)a.window;

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
        bounds[1][wave] = hi_least;
        bounds[2][wave] = lo_most;
        bounds[3][wave] = lo_least;
    }
    if (tid < 3) flags[tid] = 0;
    __syncthreads();
    int32_t all_hi = bounds[0][0], each_hi = bounds[1][0], each_lo = bounds[2][0], all_lo = bounds[3][0];
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

    const int32_t* table = a.tables + tile.run * a.table_stride;
    const uint8_t* k_base = a.cache.k + tile.kv * a.cache.head_stride;
    const uint8_t* v_base = a.cache.v + tile.kv * a.cache.head_stride;
    const int32_t last = all_hi - 1;

    // What a thread brings of a step: pieces of 16 bytes of a key, units of 4 keys and 4
    // dimensions, and (the first threads) a group's scales.
    auto piece_key = [&](int i) { return (tid + i * kThreads) / (D * kEl / 16); };
    auto piece_at = [&](int i) { return (tid + i * kThreads) % (D * kEl / 16); };
    auto unit_keys = [&](int i) { return (tid + i * kThreads) / (D / 4); };
    auto unit_dims = [&](int i) { return (tid + i * kThreads) % (D / 4); };
    struct Pages {
        int32_t k[kKLoads], v[kVLoads], group;
        uint32_t k_in[kKLoads], v_in[kVLoads], group_in;
    };
    auto page_of = [&](int32_t key, int32_t* page, uint32_t* in_page) {
        const uint32_t at = a.cache.page.div((uint32_t)min(key, last));
        *page = table[at];
        *in_page = (uint32_t)min(key, last) - at * a.cache.page.d;
    };
    auto pages_of = [&](uint32_t step) {
        Pages p;
        const int32_t key0 = (int32_t)(step * kKeys);
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) page_of(key0 + piece_key(i), &p.k[i], &p.k_in[i]);
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) page_of(key0 + 4 * unit_keys(i), &p.v[i], &p.v_in[i]);
        page_of(key0 + 8 * (tid < kGroups ? tid : 0), &p.group, &p.group_in);
        return p;
    };
    auto in_cache = [&](int32_t page) { return (uint32_t)page < a.cache.n_pages; };
    auto place_of = [&](int32_t page, uint32_t in_page) {
        return (in_cache(page) ? (int64_t)page * a.cache.page_stride : 0) + (int64_t)in_page * a.cache.token_stride;
    };
    struct Raw {
        u32x4 k[kKLoads];
        uint32_t v[kVLoads][4][kEl];
        float k_scale, v_scale;
    };
    auto load = [&](const Pages& p, Raw& r) {
#pragma unroll
        for (int i = 0; i < kKLoads; ++i)
            if (kKPieces % kThreads == 0 || tid + i * kThreads < kKPieces)
                r.k[i] = *reinterpret_cast<const u32x4*>(k_base + place_of(p.k[i], p.k_in[i]) + piece_at(i) * 16);
#pragma unroll
        for (int i = 0; i < kVLoads; ++i)
            if (kVUnits % kThreads == 0 || tid + i * kThreads < kVUnits) {
                // a unit past the row's keys begins inside them: its page has all four
                const uint8_t* v = v_base + place_of(p.v[i], p.v_in[i] & ~3u) + unit_dims(i) * 4 * kEl;
#pragma unroll
                for (int j = 0; j < 4; ++j) attn::load<4 * kEl, false>(v + j * a.cache.token_stride, r.v[i][j]);
            }
        if constexpr (E == kI8)
            if (tid < kGroups) {
                const int64_t at = (in_cache(p.group) ? p.group : 0) * a.scales.page_stride +
                                   (int64_t)(p.group_in >> a.scales.shift) * a.scales.block_stride + tile.kv * a.scales.head_stride;
                r.k_scale = a.scales.k[at];
                r.v_scale = a.scales.v[at];
            }
    };
    auto v_swizzle = [](int dim) { return kKeys == 64 ? (dim ^ (dim >> 3)) & 7 : ((dim >> 1) ^ (dim >> 3)) & 3; };
    auto store = [&](const Pages& p, Raw& r, uint32_t step, int buf, int flag) {
        const int32_t key0 = (int32_t)(step * kKeys);
        const bool partial = key0 < each_lo || key0 + kKeys > each_hi;
#pragma unroll
        for (int i = 0; i < kKLoads; ++i)
            if (kKPieces % kThreads == 0 || tid + i * kThreads < kKPieces) {
                const int key = piece_key(i), at = piece_at(i);
                const int r_lds = (key & ~12) | (key & 4) << 1 | (key & 8) >> 1;
                uint8_t* to_row = k_lds[buf] + r_lds * kKRow;
                const int by = r_lds & 7;
                if constexpr (E == kHalf) {
                    *reinterpret_cast<u32x4*>(to_row + ((at ^ by) * 16)) = r.k[i];
                } else {
                    const u32x4 w = r.k[i];
                    *reinterpret_cast<u32x4*>(to_row + (((2 * at) ^ by) * 16)) =
                        u32x4{from_byte<T, E, false>(w[0]), from_byte<T, E, true>(w[0]), from_byte<T, E, false>(w[1]), from_byte<T, E, true>(w[1])};
                    *reinterpret_cast<u32x4*>(to_row + (((2 * at + 1) ^ by) * 16)) =
                        u32x4{from_byte<T, E, false>(w[2]), from_byte<T, E, true>(w[2]), from_byte<T, E, false>(w[3]), from_byte<T, E, true>(w[3])};
                }
            }
#pragma unroll
        for (int i = 0; i < kVLoads; ++i)
            if (kVUnits % kThreads == 0 || tid + i * kThreads < kVUnits) {
                const int kg = unit_keys(i), quad = unit_dims(i);
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
                    if (partial || !in_cache(p.v[i])) {
                        const int32_t key = key0 + 4 * kg;
                        const bool paged = in_cache(p.v[i]);
                        const u32x2 keep = {(paged && key <= last ? 0xFFFFu : 0) | (paged && key + 1 <= last ? 0xFFFF0000u : 0),
                                            (paged && key + 2 <= last ? 0xFFFFu : 0) | (paged && key + 3 <= last ? 0xFFFF0000u : 0)};
                        uint32_t bad = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[e] &= keep;
                            bad |= not_finite<P>(v[e][0]) | not_finite<P>(v[e][1]);
                        }
                        if (bad) atomicOr(&flags[flag], 2u);
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int dim = 4 * quad + e;
                    *reinterpret_cast<u32x2*>(v_lds[buf] + dim * kVRow + (((kg >> 1) ^ v_swizzle(dim)) * 16) + (kg & 1) * 8) = v[e];
                }
            }
        if (tid < kGroups) {
            const bool paged = in_cache(p.group);
            f32x4 g = {a.scale, 0, 1, paged ? 1.0f : 0.0f};
            if constexpr (E == kI8) {
                const float k = a.scale * r.k_scale, v = r.v_scale;
                g[0] = k < 1e-37f ? 1e-37f : k;  // -inf times 0 is NaN
                const float up = v < 8.673617379884035e-19f ? 8.673617379884035e-19f : v;  // 2^-60
                g[1] = __builtin_amdgcn_logf(up);
                g[2] = 1.0f / up;
            }
            group_lds[buf][tid] = g;
            if (!paged && key0 + 8 * tid <= last) atomicOr(&flags[flag], 1u);
        }
    };

    f32x16 acc[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0;
    float m = -INFINITY, l = 0;

    auto v_at = [&](int buf, int dim, int slot) { return v_lds[buf] + dim * kVRow + ((slot ^ v_swizzle(dim)) * 16); };
    // Values without a number in a step that not every row sees whole: their dimension is NaN for
    // the rows that see them, and they are taken out for the others.  Rare, and slow.
    auto part_ways = [&](uint32_t step, int buf) {
        const int32_t key0 = (int32_t)(step * kKeys);
        for (int key = 0; key < kKeys; ++key) {
            const bool seen = key0 + key >= lo && key0 + key < hi && group_lds[buf][key / 8][3] != 0;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int dim = 32 * t + 8 * (i >> 2) + 4 * half + (i & 3);
                    const uint32_t v = *reinterpret_cast<const uint16_t*>(v_at(buf, dim, key / 8) + key % 8 * 2);
                    if (seen && not_finite<P>(v)) acc[t][i] = __uint_as_float(0x7FC00000u);
                }
        }
        __syncthreads();
        for (int i = tid; i < D * kVRow / 4; i += kThreads) {
            uint32_t* v = reinterpret_cast<uint32_t*>(v_lds[buf]) + i;
            *v &= ~not_finite<P>(*v);
        }
        __syncthreads();
    };

    auto compute = [&](uint32_t step, int buf, uint32_t said) {
        const int32_t key0 = (int32_t)(step * kKeys);
        if (key0 >= hi_most || key0 + kKeys <= lo_least) return;
        f32x16 sc[kSub];
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[u][i] = 0;
            const uint8_t* k_row = k_lds[buf] + (32 * u + col) * kKRow;
#pragma unroll
            for (int st = 0; st < kSteps; ++st)
                sc[u] = mfma32(T{}, *reinterpret_cast<const u32x4*>(k_row + (((2 * st + half) ^ (col & 7)) * 16)), qf[st], sc[u]);
        }
        f32x4 group[2 * kSub];
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) group[j] = E == kI8 ? group_lds[buf][2 * j + half] : f32x4{a.scale, 0, 1, 1};
        if (key0 < lo_most || key0 + kKeys > hi_least || (said & 1)) {
#pragma unroll
            for (int j = 0; j < 2 * kSub; ++j) {
                const bool paged = group_lds[buf][2 * j + half][3] != 0;
                const int32_t key = key0 + 16 * j + 8 * half;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool seen = paged && key + i >= lo && key + i < hi;
                    sc[j / 2][8 * (j & 1) + i] = seen ? sc[j / 2][8 * (j & 1) + i] : -INFINITY;
                }
                // nor are the scales of a group that the row does not see
                if (E == kI8 && !(paged && key + 8 > lo && key < hi)) group[j] = f32x4{1, 0, 0, 0};
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
        const float lift = P::base_of(halves_max(top));
        if (__any(lift > m)) {
            const float up = fmaxf(m, lift), by = exp2_of(m - above(up));
            m = up;
            l *= by;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) acc[t] *= by;
        }
        const float base = above(m);
        constexpr float kUp = 549755813888.0f;  // 2^39
        bool low = false;
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
            const float off = E == kI8 ? group[j][1] - base : -base, by = E == kI8 ? group[j][0] : a.scale;
            float sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = exp2_of(__builtin_fmaf(sc[j / 2][8 * (j & 1) + i], by, off));
                sc[j / 2][8 * (j & 1) + i] = s;
                sum += s;
                if constexpr (kLow) low = low || (s < 0.25f && s > 0);
            }
            l = E == kI8 ? __builtin_fmaf(sum, group[j][2], l) : l + sum;
        }
        auto add = [&](int j, u32x4 pf) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                acc[t] = mfma32(P{}, *reinterpret_cast<const u32x4*>(v_at(buf, 32 * t + col, 2 * j + half)), pf, acc[t]);
        };
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = sc[j / 2][8 * (j & 1) + i];
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                u32x4 pf;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    pf[i / 2] = P::pair(p[i], p[i + 1]);
                    if (kParts > 1) {
                        p[i] -= P::low(pf[i / 2]);
                        p[i + 1] -= P::high(pf[i / 2]);
                    }
                }
                add(j, pf);
            }
            if constexpr (kLow) {
                if (!__any(low)) continue;
                // what two parts leave of p < 2^-2, 2^39 up
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = sc[j / 2][8 * (j & 1) + i] < 0.25f ? p[i] * kUp : 0.0f;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) acc[t] *= kUp;
#pragma unroll
                for (int k = 0; k < kParts; ++k) {
                    u32x4 pf;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        pf[i / 2] = P::pair(p[i], p[i + 1]);
                        p[i] -= P::low(pf[i / 2]);
                        p[i + 1] -= P::high(pf[i / 2]);
                    }
                    add(j, pf);
                }
#pragma unroll
                for (int t = 0; t < kTiles; ++t) acc[t] *= 1.0f / kUp;
            }
        }
    };

    if (from < to) {
        Raw raw;
        Pages now = pages_of(from);
        load(now, raw);
        Pages then = pages_of(min(from + 1, to - 1));
        store(now, raw, from, 0, 0);
        __syncthreads();
        int flag = 0;
        for (uint32_t step = from; step < to; ++step) {
            const int buf = (int)(step - from) & 1, next_flag = flag == 2 ? 0 : flag + 1;
            const bool more = step + 1 < to;
            if (more) {
                now = then;
                load(now, raw);
                then = pages_of(min(step + 2, to - 1));
            }
            const uint32_t said = flags[flag];
            if constexpr (E != kI8)
                if (said & 2) part_ways(step, buf);
            compute(step, buf, said);
            if (more) store(now, raw, step + 1, buf ^ 1, next_flag);
            // the flags of the step after the next: read last a step ago, before a barrier
            if (tid == 0) flags[next_flag == 2 ? 0 : next_flag + 1] = 0;
            flag = next_flag;
            __syncthreads();
        }
    }

    l = halves_sum(l);
    if (!real) return;
    if (a.splits > 1) {
        const int64_t entry = (((int64_t)slot * a.by_units.d + unit) * a.splits + blockIdx.y) * (W * kWaveRows) + at_row;
        float* o = a.part_acc + entry * D + 4 * half;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(o + 32 * t + 2 * i) = f32x4{acc[t][i], acc[t][i + 1], acc[t][i + 2], acc[t][i + 3]};
        if (half == 0) a.part_ml[entry] = make_float2(m, l);
        return;
    }
    const float over = l > 0 || l != l ? a.cache.v_scale / l : 0.0f;
    uint8_t* out = a.out + row * a.out_stride + (int64_t)head * D * (kF32 ? 4 : 2);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        if constexpr (kF32) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(out + (32 * t + 2 * i + 4 * half) * 4) =
                    f32x4{acc[t][i], acc[t][i + 1], acc[t][i + 2], acc[t][i + 3]} * over;
        } else {
            // the two lanes of a column exchange fours: dimensions 0 - 7 to one, 8 - 15 to the other
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) w[e / 2] = T::pair(acc[t][i + e] * over, acc[t][i + e + 1] * over);
                const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                *reinterpret_cast<u32x4*>(out + (32 * t + 2 * i + 8 * half) * 2) = u32x4{x[0], y[0], x[1], y[1]};
            }
        }
    }
    if (a.lse && half == 0) a.lse[(int64_t)row * a.q_heads + head] = log_sum(m, l);
}

template <int D, class T, Elem E>
hipError_t launch_prompt_elem(const PromptArgs& a, bool out_f32, hipStream_t s) {
    const dim3 grid(a.tiles * a.by_units.d, a.splits), block(64 * prompt_waves(D));
    if (out_f32)
        hipLaunchKernelGGL((prompt_kernel<D, T, E, true>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((prompt_kernel<D, T, E, false>), grid, block, 0, s, a);
    return hipGetLastError();
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
