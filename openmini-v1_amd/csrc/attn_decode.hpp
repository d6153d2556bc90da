// Attention of single query tokens over a paged cache (openmini_attn_decode).
//
// A row's query heads that share a key head are the columns of 16 x 16 MFMA tiles.  For each
// 32 keys a wave computes
//   S^T = K q^T   (two 16-key tiles, head_dim in steps of 32)
//   p = 2^(s - m), m and l the running maximum and sum of each column (s in powers of two)
//   O^T += V^T P^T (head_dim in tiles of 16, all 32 keys at once)
// The C layout of S^T gives lane (g = lane / 16, column lane % 16) rows 4 g .. 4 g + 3 of
// each tile, and the B layout of P^T wants k = 8 g .. 8 g + 7 of the column in the same
// lane.  With row r of tile s being key 8 (r / 4) + 4 s + r % 4, the two are the same keys:
// the probabilities go from one product to the next without leaving their lane, the running
// maximum scales the accumulators without a broadcast, and a lane's keys are eight
// neighbours, which share a page.
//
// V^T's A layout wants eight keys of one dimension in a lane.  A lane loads head_dim / 16
// neighbouring dimensions of each of its eight keys (a row of the cache is read by 16
// neighbouring lanes, whole) and transposes them in registers, two keys to a dword, one
// byte permutation each; tile e of a chunk is then dimensions e, e + width, ...
//
// The probabilities enter the second product as the sum of three bf16 or two fp16 parts (fp16
// caches), together all of fp32 or nearly: their rounding to one bf16 would be 2^-9 of an fp32
// output, to two 2^-18 (1.2e-6 measured, against 4e-7 for fp32 arithmetic throughout).  bf16 has
// the range of fp32.  fp16 has a least unit of 2^-24, so there p is 2^15 at the maximum, and
// where a tile has keys whose two parts hold less than 22 bits (p below 2^-17 of the largest: a
// first key that draws most of the weight leaves the others there), what the two leave is
// added too, as two parts 2^39 up.  Sums, maxima and the joined parts are fp32.
//
// Bound by memory: one operation a byte (e4m3: two) for each query head of a key head.  A tile
// of 32, 64 or 128 keys is about 16 KB; the loads of the next tile are issued as soon as the
// registers of the present one are free, one wave to a SIMD, a row's first behind the last
// products of the row before.  Measured (MI355X, us with the second launch, which is 4 to 6
// of them; in brackets a read of as many bytes): 131071 keys of one row, 8 heads of 128, bf16
// 90 (83), the kernel alone 84, 6.4 TB/s; 16 rows of 700 - 2100 keys, 32 heads of 128, fp16 53
// (50); 64 rows of up to 4096 keys in a window, 4 heads of 64, bf16 28 (17); 128 rows of 2000 -
// 12000 keys, 8 heads of 128, e4m3 245 (230).  One row of 300 keys, in one launch, 7.1 (2.4, a
// launch).  Heads of 64 in e4m3 are bound by the issue of instructions instead (195 vector
// instructions for 32 keys): 100 rows of 1000 - 8000 keys, 8 heads, 85 us, 4.3 TB/s.
#pragma once

#include <type_traits>

#include "attn_internal.hpp"
#include "qmm_device.hpp"

namespace attn {

using qmm::bf16x8;
using qmm::f16x8;
using qmm::f32x4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct BF16 {
    static constexpr int kExactParts = 3;  // that hold an fp32 probability, 8 bits each
    static constexpr bool kNarrow = false;  // parts have the range of fp32
    // The base m of p = 2^(s - m) for a largest s.
    static __device__ __forceinline__ float base_of(float top) { return top; }
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(__bf16)a, (__bf16)b});
    }
    static __device__ __forceinline__ float low(uint32_t u) { return __uint_as_float(u << 16); }
    static __device__ __forceinline__ float high(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }
    template <bool kHigh>
    static __device__ __forceinline__ uint32_t from_f8(uint32_t u) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, kHigh));
    }
};

struct F16 {
    static constexpr int kExactParts = 2;  // 11 bits each, for p from 2^-2 on
    static constexpr bool kNarrow = true;
    // p of at most 2^15, below the largest fp16.  From 2^23 on the difference need not be
    // exact and could round to 2^16: there p is at most 1, and scores are 1 apart at least.
    static __device__ __forceinline__ float base_of(float top) { return fabsf(top) < 8388608.0f ? top - 15.0f : top; }
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        return __builtin_bit_cast(uint32_t, qmm::f16x2{(_Float16)a, (_Float16)b});
    }
    static __device__ __forceinline__ float low(uint32_t u) { return (float)__builtin_bit_cast(qmm::f16x2, u)[0]; }
    static __device__ __forceinline__ float high(uint32_t u) { return (float)__builtin_bit_cast(qmm::f16x2, u)[1]; }
    template <bool kHigh>
    static __device__ __forceinline__ uint32_t from_f8(uint32_t u) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, kHigh));
    }
};

// kStream: loads that leave the caches to others (decode_streams).
template <bool kStream, class V>
__device__ __forceinline__ V load_as(const uint8_t* p) {
    if constexpr (kStream) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    return *reinterpret_cast<const V*>(p);
}
template <int kBytes, bool kStream>
__device__ __forceinline__ void load(const uint8_t* p, uint32_t* d) {
    if constexpr (kBytes == 16) {
        const u32x4 v = load_as<kStream, u32x4>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = v[i];
    } else if constexpr (kBytes == 8) {
        const u32x2 v = load_as<kStream, u32x2>(p);
        d[0] = v[0];
        d[1] = v[1];
    } else if constexpr (kBytes == 4) {
        d[0] = load_as<kStream, uint32_t>(p);
    } else {
        d[0] = load_as<kStream, uint16_t>(p);
    }
}

// Inclusive prefix sum over the wave.
__device__ __forceinline__ uint32_t wave_sums(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
    return v;
}

// Over the four lanes of a column (lane % 16): every one of them gets the maximum (sum).
__device__ __forceinline__ float column_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}


// 2^(a - m) for a maximum m that is -inf where nothing is seen.
__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ float exp2_of(float a) { return __builtin_amdgcn_exp2f(a); }

struct Span {
    int32_t lo, hi;   // the keys that a row sees
    uint32_t tiles;
    __device__ __forceinline__ uint32_t weight() const { return max(tiles, 1u); }
};

// What a wave needs first.  These are kernel arguments of their own, in front: the first 14
// dwords of them are in SGPRs when a wave starts, while the others are still to be loaded.
struct First {
    const int32_t *lens, *rows;
    uint32_t n_rows, requests, max_len, window, shares;
    uint32_t uncut;  // the shares are rows (decode_uncut)
};

// What the call says of a row, and the same by scalar loads (a uniform row; they are not
// counted with a wave's loads of keys and values, and wait for none of them).
struct Said {
    int32_t keys, request;
};
__device__ __forceinline__ Said said_of(const First& a, uint32_t r) {
    return {a.lens[r], a.rows ? a.rows[r] : (int32_t)r};
}
typedef const __attribute__((address_space(4))) int32_t ConstInt;
__device__ __forceinline__ Said said_of_uniform(const First& a, uint32_t r) {
    return {((ConstInt*)a.lens)[r], a.rows ? ((ConstInt*)a.rows)[r] : (int32_t)r};
}

// No keys for a request outside the tables.
template <uint32_t kKeys>
__device__ __forceinline__ Span span_of(const First& a, Said said) {
    Span s;
    s.hi = min(max(said.keys, 0), (int32_t)a.max_len);
    if ((uint32_t)said.request >= a.requests) s.hi = 0;
    s.lo = (int32_t)max((uint32_t)s.hi, a.window) - (int32_t)a.window;  // window: at least 1
    s.tiles = ((uint32_t)s.hi + kKeys - 1) / kKeys - (uint32_t)s.lo / kKeys;
    return s;
}

// Where a wave starts.  The tiles of all rows stand in one line (a row without keys takes
// the place of one, for its zeros to be written); share p of it is [p each, (p + 1) each),
// whatever rows that is.  So every share is as long as every other, however the lengths
// differ.
struct Share {
    uint32_t each, from, to;  // tiles of a share; this one's place in the line
    uint32_t row, row_at;     // its first row, and that row's place
};

template <uint32_t kKeys, int W>
__device__ __forceinline__ bool find_share(const First& a, uint32_t p, Share& out, Said& said) {
    const uint32_t lane = threadIdx.x & 63;
    auto place = [&](uint32_t total) {
        out.each = (total + a.shares - 1) / a.shares;
        out.from = min(p * out.each, total);  // below 2^32: total < 2^31, p < 2 shares but for few tiles
        out.to = min(out.from + out.each, total);
        return out.from < total;
    };
    if (a.uncut) {  // rows are its places
        if (!place(a.n_rows)) return false;
        out.row = out.row_at = out.from;
        said = said_of_uniform(a, out.row);
        return true;
    }
    if (a.n_rows <= 64) {  // every wave by itself
        Said mine = {0, 0};
        Span s = {0, 0, 0};
        uint32_t n = 0;
        if (lane < a.n_rows) {
            mine = said_of(a, lane);
            s = span_of<kKeys>(a, mine);
            n = s.weight();
        }
        const uint32_t upto = wave_sums(n);
        if (!place((uint32_t)__builtin_amdgcn_readlane((int)upto, 63))) return false;
        const int at = __ffsll((unsigned long long)__ballot(out.from >= upto - n && out.from < upto)) - 1;
        out.row = (uint32_t)at;
        out.row_at = (uint32_t)__builtin_amdgcn_readlane((int)(upto - n), at);
        said.keys = __builtin_amdgcn_readlane(s.hi, at);
        said.request = __builtin_amdgcn_readlane(mine.request, at);
        return true;
    }
    // each thread sums some rows; the one whose rows pass a wave's start looks through them
    __shared__ uint32_t wave_total[W], start[W], found[W][2];
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t each = (a.n_rows + 64 * W - 1) / (64 * W);
    const uint32_t r0 = min(threadIdx.x * each, a.n_rows), r1 = min(r0 + each, a.n_rows);
    uint32_t n = 0;
    for (uint32_t r = r0; r < r1; ++r) n += span_of<kKeys>(a, said_of(a, r)).weight();
    uint32_t upto = wave_sums(n);
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t w = 0; w < W; ++w) {
        if (w == wave) upto += total;
        total += wave_total[w];
    }
    const bool any = place(total);
    if (lane == 0) start[wave] = out.from;
    __syncthreads();
    for (uint32_t w = 0; w < W; ++w) {
        const uint32_t from = start[w];
        if (from >= upto - n && from < upto) {
            uint32_t at = upto - n, r = r0;
            for (; r + 1 < r1; ++r) {
                const uint32_t weight = span_of<kKeys>(a, said_of(a, r)).weight();
                if (from < at + weight) break;
                at += weight;
            }
            found[w][0] = r;
            found[w][1] = at;
        }
    }
    __syncthreads();
    if (!any) return false;
    out.row = (uint32_t)__builtin_amdgcn_readfirstlane((int)found[wave][0]);
    out.row_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)found[wave][1]);
    said = said_of_uniform(a, out.row);
    return true;
}

// kWide: a key's place in the cache takes 64 bits (caches of 4 GiB and more); else 32, which
// the loads add to a scalar address by themselves.
// kWhole: a workgroup takes a row of one unit, its waves equal runs of the row's tiles, and
// they are joined in LDS: one launch, and no wave that looks for its share, but as many CUs
// as there are rows and units, and a CU reads about 50 GB/s.  For short rows (decode_whole);
// the last tile of a wave is most of its work then, so no loads of a next one are behind it.
template <int D, class T, bool F8, int kSub, int W, bool kWide, bool kWhole, bool kStream>
__global__ __launch_bounds__(64 * W, D == 256 && !F8 ? 1 : 2) void decode_kernel(const int32_t* lens, const int32_t* rows,
                                                                                 uint32_t n_rows, uint32_t requests,
                                                                                 uint32_t max_len, uint32_t window,
                                                                                 uint32_t shares, uint32_t units,
                                                                                 uint32_t units_m, uint32_t units_shift, uint32_t eighth,
                                                                                 uint32_t uncut,
                                                                                 DecodeArgs a) {
    const First f = {lens, rows, n_rows, requests, max_len, window, shares, uncut};
    using P = std::conditional_t<F8, BF16, T>;  // of the second product's parts: both hold e4m3
    constexpr int kEl = F8 ? 1 : 2;           // bytes of a cache element
    constexpr uint32_t kKeys = 32 * kSub;     // keys of a tile, in kSub tiles of 32
    constexpr int kSteps = D / 32;            // MFMAs over head_dim of the first product
    constexpr int kTiles = D / 16;            // 16-dimension tiles of the second
    constexpr int kKWords = kSteps * 2 * kEl; // dwords of a key in a lane
    constexpr int kVWords = (kTiles * kEl + 3) / 4;
    // V in chunks of 128, 64 and 32 dimensions, of which a lane holds 8, 4 and 2
    constexpr int kFull = D / 128, kRest = D % 128;
    constexpr bool kHas64 = kRest >= 64, kHas32 = kRest % 64 != 0;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;

    // Waves in line: the units (key heads, or tiles of their query heads) of share 0, of
    // share 1, ...; workgroups go round the 8 XCDs by index, and each XCD takes one eighth of
    // the line.  So the heads of a share run side by side: in a cache of
    // [tokens][heads][dims] they read whole stretches of memory together (537 MB of keys and
    // values in bf16, heads of 128, loads alone: 88 us; a workgroup to a head: 95 us).
    const uint32_t line = (blockIdx.x & 7) * eighth + (blockIdx.x >> 3);
    const uint32_t w_no = line * W + (uint32_t)wave;
    const uint32_t at = kWhole ? line : w_no;  // share_no: the row, kWhole
    const uint32_t share_no = units_m ? __umulhi(at, units_m) >> units_shift : at, unit = at - share_no * units;
    const uint32_t kv = a.by_head_tiles.div(unit), head_tile = unit - kv * (uint32_t)a.head_tiles;
    Share share;
    Said said;
    if constexpr (kWhole) {
        if (share_no >= n_rows) return;
        said = said_of_uniform(f, share_no);
        const uint32_t weight = span_of<kKeys>(f, said).weight();
        share.each = (weight + W - 1) / W;
        share.from = min(share.each * wave, weight);
        share.to = min(share.from + share.each, weight);
        share.row = share_no;
        share.row_at = 0;
    } else if (!find_share<kKeys, W>(f, share_no, share, said)) {
        if (!a.by_row && unit == 0 && share_no < shares && lane == 0) a.split[share_no] = Split{0, 0, 0};
        return;
    }
    const int heads = min(kHeadTile, a.group - (int)head_tile * kHeadTile);  // columns in use
    const int head0 = (int)kv * a.group + (int)head_tile * kHeadTile;

    // A row's stretch of the share: tiles [tile0, tile1) of its keys [lo, hi).
    struct Row {
        uint32_t row, at, end;  // its places in the line: [at, end)
        uint32_t tile0, tile1;
        int32_t lo, hi;
        const int32_t* table;
    };
    auto row_of = [&](uint32_t row, uint32_t at, uint32_t from, Said said) {
        const Span s = span_of<kKeys>(f, said);
        Row r;
        r.row = row;
        r.at = at;
        r.end = at + (f.uncut ? 1 : s.weight());
        r.tile0 = (uint32_t)s.lo / kKeys + (from - at);
        r.tile1 = f.uncut ? r.tile0 + s.tiles : s.tiles ? (uint32_t)s.lo / kKeys + (min(r.end, share.to) - at) : r.tile0;
        r.lo = s.lo;
        r.hi = s.hi;
        r.table = a.tables + (int64_t)said.request * a.table_stride;
        return r;
    };

    // q^T: lane holds column `col`, eight dimensions a step, in the order of a key's loads;
    // columns past the heads in use hold the last of them again
    u32x4 qf[kSteps];
    auto load_q = [&](uint32_t row) {
        const uint8_t* q = a.q + row * a.q_stride + (int64_t)(head0 + min(col, heads - 1)) * D * 2;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const int dim = F8 && (st | 1) < kSteps ? (st >> 1) * 64 + g * 16 + (st & 1) * 8 : st * 32 + g * 8;
            qf[st] = *reinterpret_cast<const u32x4*>(q + dim * 2);
        }
    };

    const uint8_t* k_base = a.cache.k + kv * a.cache.head_stride;
    const uint8_t* v_base = a.cache.v + kv * a.cache.head_stride;
    const int kg = col >> 2, k_row = col & 3;  // the lane's key of tile s: 8 kg + 4 s + k_row

    // A tile of some row; the eight keys from 8 * grp of its 32 `sub` on, kept inside the
    // row's keys; the column of their page, and their place in the cache.
    struct Tile {
        uint32_t no;
        int32_t first_group, last_group;
        const int32_t* table;
    };
    auto tile_of = [](const Row& r, uint32_t no) { return Tile{no, r.lo & ~7, (r.hi - 1) & ~7, r.table}; };
    auto group_at = [&](const Tile& t, int sub, int grp) -> int32_t {
        return min(max((int32_t)(t.no * kKeys) + 32 * sub + 8 * grp, t.first_group), t.last_group);
    };
    // Eight keys of a tile, for all its groups.
    auto one_group = [&](const Row& r, uint32_t no) {
        Tile t = tile_of(r, no);
        t.first_group = t.last_group = min(max((int32_t)(no * kKeys), t.first_group), t.last_group);
        return t;
    };
    using Place = std::conditional_t<kWide, uint64_t, uint32_t>;
    struct Pages {  // of a tile's K and V groups, and the groups' places in them
        int32_t k[kSub], v[kSub];
        uint32_t k_in[kSub], v_in[kSub];
    };
    auto page_of = [&](const Tile& t, int32_t key, int32_t* page, uint32_t* in_page) {
        const uint32_t at = a.cache.page.div_by_many((uint32_t)key);
        *page = t.table[at];
        *in_page = (uint32_t)key - at * a.cache.page.d;
    };
    auto pages_of = [&](const Tile& t) {
        Pages p;
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            page_of(t, group_at(t, u, kg), &p.k[u], &p.k_in[u]);
            page_of(t, group_at(t, u, g), &p.v[u], &p.v_in[u]);
        }
        return p;
    };
    auto place_of = [&](int32_t page, uint32_t in_page) -> Place {
        return ((uint32_t)page < a.cache.n_pages ? (Place)(uint32_t)page * (Place)a.cache.page_stride : 0) +
               (Place)in_page * (Place)a.cache.token_stride;
    };

    uint32_t kraw[kSub][2][kKWords], vraw[kSub][8][kVWords];
    auto load_k = [&](const Pages& pages) {
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            const Place at = place_of(pages.k[u], pages.k_in[u] + k_row) + g * 16;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint8_t* p = k_base + 4 * s * a.cache.token_stride;
                if constexpr (F8) {
#pragma unroll
                    for (int c = 0; c < kSteps / 2; ++c) load<16, kStream>(p + at + c * 64, &kraw[u][s][4 * c]);
                    if constexpr (kSteps & 1) load<8, kStream>(p + (at - g * 8) + (kSteps - 1) * 32, &kraw[u][s][2 * (kSteps - 1)]);
                } else {
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) load<16, kStream>(p + at + st * 64, &kraw[u][s][4 * st]);
                }
            }
        }
    };
    auto load_v = [&](const Pages& pages, int u) {
        const Place at = place_of(pages.v[u], pages.v_in[u]);
        const Place at128 = at + col * 8 * kEl, at64 = at + col * 4 * kEl, at32 = at + col * 2 * kEl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t* p = v_base + j * a.cache.token_stride;
#pragma unroll
            for (int c = 0; c < kFull; ++c) load<8 * kEl, kStream>(p + at128 + c * 128 * kEl, &vraw[u][j][c * 2 * kEl]);
            if constexpr (kHas64) load<4 * kEl, kStream>(p + at64 + kFull * 128 * kEl, &vraw[u][j][kFull * 2 * kEl]);
            if constexpr (kHas32)
                load<2 * kEl, kStream>(p + at32 + (kFull * 128 + kHas64 * 64) * kEl, &vraw[u][j][kFull * 2 * kEl + kHas64 * kEl]);
        }
    };

    Pages now, then;  // of the present tile and the next
    f32x4 acc[kTiles], sc[kSub][2];
    float m, l;
    auto scores = [&] {
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                sc[u][s] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                    u32x4 kf;
                    if constexpr (F8) {
                        const uint32_t w0 = kraw[u][s][2 * st], w1 = kraw[u][s][2 * st + 1];
                        kf = u32x4{T::template from_f8<false>(w0), T::template from_f8<true>(w0),
                                   T::template from_f8<false>(w1), T::template from_f8<true>(w1)};
                    } else {
                        kf = u32x4{kraw[u][s][4 * st], kraw[u][s][4 * st + 1], kraw[u][s][4 * st + 2],
                                   kraw[u][s][4 * st + 3]};
                    }
                    sc[u][s] = T::mfma(kf, qf[st], sc[u][s]);
                }
            }
    };
    auto outputs = [&](const Row& cur, uint32_t tile, auto next_tag) {
        // keys outside the row's or on no page of the cache: only a row's first and
        // last tiles, and broken tables, have them
        float x[kSub][8], least = INFINITY;  // least before the mask: a tile's edge is not low
        const int32_t key0 = (int32_t)(tile * kKeys) + 8 * g;
        bool whole = key0 >= cur.lo && key0 + (int32_t)kKeys - 24 <= cur.hi;
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[u][j] = sc[u][j / 4][j % 4] * a.scale;
                if constexpr (P::kNarrow) least = fminf(least, x[u][j]);
            }
            whole = whole && (uint32_t)now.v[u] < a.cache.n_pages;
        }
        if (!__all(whole)) {
#pragma unroll
            for (int u = 0; u < kSub; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int32_t key = key0 + 32 * u + j;
                    const bool seen = (uint32_t)now.v[u] < a.cache.n_pages && key >= cur.lo && key < cur.hi;
                    x[u][j] = seen ? x[u][j] : -INFINITY;
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) vraw[u][j][w] = seen ? vraw[u][j][w] : 0;  // 0 * NaN is NaN
                }
        }
        float top = x[0][0];
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, x[u][j]);
        const float lift = P::base_of(column_max(top)), to = fmaxf(m, lift), base = above(to);
        constexpr float kUp = 549755813888.0f;  // 2^39
        bool low = false;
        if constexpr (P::kNarrow) low = __any(least < base - 2.0f);
        if (low || __any(lift > m)) {
            float by = exp2_of(m - base);
            m = to;
            l *= by;
            if (low) by *= kUp;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) acc[i] *= by;
        }
        // second product, p as the sum of kParts 16-bit parts
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            constexpr int kParts = P::kExactParts;
            u32x4 pf[kParts];
            auto split = [&](float r0, float r1, int j) {
#pragma unroll
                for (int k = 0; k < kParts; ++k) {
                    const uint32_t h = P::pair(r0, r1);
                    pf[k][j / 2] = h;
                    r0 -= P::low(h);
                    r1 -= P::high(h);
                }
                return make_float2(r0, r1);
            };
            // a low tile's first time round: what the parts leave of p < 2^-2, at most 2^-25, is
            // added to the accumulators 2^39 up.  All tiles low against none: 131071 keys of one
            // row 90.4 / 90.3 us, 64 rows of heads of 64 31.0 / 29.9, one row of 300 keys 8.2 / 7.4.
            for (bool rest = low;; rest = false) {
                if (rest) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float r0 = exp2_of(x[u][j] - base), r1 = exp2_of(x[u][j + 1] - base);
                        const float2 r = split(r0, r1, j);
                        split(r0 < 0.25f ? r.x * kUp : 0.0f, r1 < 0.25f ? r.y * kUp : 0.0f, j);
                    }
                    if (u > 0)
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) acc[t] *= kUp;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float r0 = exp2_of(x[u][j] - base), r1 = exp2_of(x[u][j + 1] - base);
                        l += r0 + r1;
                        split(r0, r1, j);
                    }
                }
                // a zero that is not known to be one: else V's fragments are made before the loop
                // and kept (up to 60 registers)
                uint32_t zero = 0;
                if constexpr (P::kNarrow) asm volatile("" : "+s"(zero));
                auto add = [&](int t, u32x4 vf) {
#pragma unroll
                    for (int k = 0; k < kParts; ++k) acc[t] = P::mfma(vf, pf[k], acc[t]);
                };
                auto chunk = [&](int t0, int word0, auto width_tag) {
                    constexpr int kWidth = decltype(width_tag)::value;
                    if constexpr (F8) {
#pragma unroll
                        for (int w = 0; w < (kWidth + 3) / 4; ++w) {
                            u32x4 f[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const uint32_t v0 = vraw[u][2 * q][word0 + w], v1 = vraw[u][2 * q + 1][word0 + w];
                                const uint32_t lo = __builtin_amdgcn_perm(v1, v0, 0x05010400u);
                                f[0][q] = P::template from_f8<false>(lo);
                                f[1][q] = P::template from_f8<true>(lo);
                                if constexpr (kWidth >= 4) {
                                    const uint32_t hi = __builtin_amdgcn_perm(v1, v0, 0x07030602u);
                                    f[2][q] = P::template from_f8<false>(hi);
                                    f[3][q] = P::template from_f8<true>(hi);
                                }
                            }
#pragma unroll
                            for (int e = 0; e < (kWidth < 4 ? kWidth : 4); ++e) add(t0 + 4 * w + e, f[e]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < kWidth; ++e) {
                            u32x4 f;
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                f[q] = __builtin_amdgcn_perm(vraw[u][2 * q + 1][word0 + e / 2], vraw[u][2 * q][word0 + e / 2],
                                                             (e & 1 ? 0x07060302u : 0x05040100u) + zero);
                            add(t0 + e, f);
                        }
                    }
                };
#pragma unroll
                for (int c = 0; c < kFull; ++c) chunk(8 * c, c * 2 * kEl, std::integral_constant<int, 8>{});
                if constexpr (kHas64) chunk(8 * kFull, kFull * 2 * kEl, std::integral_constant<int, 4>{});
                if constexpr (kHas32)
                    chunk(8 * kFull + 4 * kHas64, kFull * 2 * kEl + kHas64 * kEl, std::integral_constant<int, 2>{});
                if (!rest) break;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) acc[t] *= 1.0f / kUp;
            }
            // the next tile's, into the registers that are free
            if constexpr (decltype(next_tag)::value) load_v(then, u);
        }
    };

    // The share's tiles, row after row.  The loads run a tile ahead and the pages two, from
    // a row into the next: a row's last products are behind the next row's first loads.
    Row cur = row_of(share.row, share.row_at, share.from, said);
    bool loaded = false;  // cur's first tile is on its way
    for (;;) {
        const bool more = !kWhole && cur.end < share.to;
        if (more) said = said_of_uniform(f, cur.row + 1);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0, 0, 0, 0};
        m = -INFINITY;
        l = 0;
        uint32_t tile = cur.tile0;
        Row following = cur;
        if (!loaded && tile < cur.tile1) {
            const Tile first = tile_of(cur, tile), second = tile + 1 < cur.tile1 ? tile_of(cur, tile + 1) : one_group(cur, tile);
            now = pages_of(first);
            load_q(cur.row);
            then = pages_of(second);
            load_k(now);
#pragma unroll
            for (int u = 0; u < kSub; ++u) load_v(now, u);
        }
        if constexpr (kWhole) {
            for (; tile + 1 < cur.tile1; ++tile) {
                scores();
                const Pages later = pages_of(tile_of(cur, min(tile + 2, cur.tile1 - 1)));
                load_k(then);
                outputs(cur, tile, std::true_type{});
                now = then;
                then = later;
            }
            if (tile < cur.tile1) {
                scores();
                outputs(cur, tile, std::false_type{});
            }
        } else {
            for (; tile + 2 < cur.tile1; ++tile) {
                scores();
                // the pages of the tile after the next, then the next keys: their pages came
                // with loads that have been waited for
                const Pages later = pages_of(tile_of(cur, tile + 2));
                load_k(then);
                outputs(cur, tile, std::true_type{});
                now = then;
                then = later;
            }
            // The row's last two tiles, before which come the next row's first.  At the share's
            // end (or before a row without keys) it is eight keys of the present one again, for
            // the whole tile: loads without a branch around them, so that the wait for the present
            // values need not cover them.
            if (more) following = row_of(cur.row + 1, cur.end, cur.end, said);
            loaded = tile < cur.tile1 && more && following.tile0 < following.tile1;
            for (; tile < cur.tile1; ++tile) {
                const bool last = tile + 1 == cur.tile1, cross = last && loaded;
                scores();
                const Tile after = loaded ? tile_of(following, min(following.tile0 + (last ? 1u : 0u), following.tile1 - 1))
                                          : one_group(cur, cur.tile1 - 1);
                const Pages later = pages_of(after);
                if (cross && cur.tile1 - cur.tile0 == 1)  // no tile before looked them up
                    then = pages_of(tile_of(following, following.tile0));
                load_k(then);
                if (cross) load_q(following.row);
                outputs(cur, tile, std::true_type{});
                if (last && !cross) break;
                now = then;
                then = later;
            }
        }

        l = column_sum(l);
        // accumulator i of tile t is dimension chunk + (4 g + i) * width + (t in the chunk): a
        // lane stores the chunk's width neighbours at a time
        auto each_run = [&](auto&& f) {
#pragma unroll
            for (int c = 0; c < kTiles;) {
                const int width = c / 8 < kFull ? 8 : kHas64 && c < 8 * kFull + 4 ? 4 : 2;
#pragma unroll
                for (int i = 0; i < 4; ++i) f(c, i, width, c * 16 + (4 * g + i) * width);
                c += width;
            }
        };
        if constexpr (kWhole) {
            // a wave past the row's tiles has seen nothing: maximum -inf, sum 0
            __shared__ __attribute__((aligned(16))) float part[W][kHeadTile][D + 4];
            __shared__ float2 part_ml[W][kHeadTile];
            if (col < heads) {
                each_run([&](int t, int i, int width, int d) {
                    float* o = &part[wave][col][d];
                    if (width >= 4) {
#pragma unroll
                        for (int e = 0; e < width; e += 4)
                            *reinterpret_cast<f32x4*>(o + e) =
                                f32x4{acc[t + e][i], acc[t + e + 1][i], acc[t + e + 2][i], acc[t + e + 3][i]};
                    } else {
                        *reinterpret_cast<float2*>(o) = make_float2(acc[t][i], acc[t + 1][i]);
                    }
                });
                if (g == 0) part_ml[wave][col] = make_float2(m, l);
            }
            __syncthreads();
            for (int at = (int)threadIdx.x; at < heads * (D / 4); at += 64 * W) {
                const int h = at / (D / 4), d = at % (D / 4) * 4;
                float2 ml[W];
                float top = -INFINITY, sum = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    ml[w] = part_ml[w][h];
                    top = fmaxf(top, ml[w].x);
                }
                f32x4 v = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float by = exp2_of(ml[w].x - above(top));
                    sum += ml[w].y * by;
                    v += *reinterpret_cast<const f32x4*>(&part[w][h][d]) * by;
                }
                v *= sum > 0 || sum != sum ? a.cache.v_scale / sum : 0.0f;
                const int64_t to = (int64_t)(head0 + h) * D + d;
                uint8_t* out = a.out + cur.row * a.out_stride;
                if (a.out_f32)
                    *reinterpret_cast<f32x4*>(out + to * 4) = v;
                else
                    *reinterpret_cast<uint2*>(out + to * 2) = make_uint2(T::pair(v[0], v[1]), T::pair(v[2], v[3]));
                if (a.lse && d == 0) a.lse[(int64_t)cur.row * a.q_heads + head0 + h] = log_sum(top, sum);
            }
            return;
        }
        // the row's shares: all but the first begin inside it
        const uint32_t row = cur.row, first_share = cur.at / share.each, parts = (cur.end - 1) / share.each - first_share + 1;
        if (a.by_row && unit == 0 && lane == 0 && share_no == first_share) a.split[row] = Split{row, first_share, parts};
        if (col < heads) {
            if (parts == 1) {
                const float over = l > 0 || l != l ? a.cache.v_scale / l : 0.0f;
                const int64_t at = (int64_t)(head0 + col) * D;
                if (a.out_f32) {
                    float* o = reinterpret_cast<float*>(a.out + row * a.out_stride) + at;
                    each_run([&](int t, int i, int width, int d) {
                        if (width >= 4) {
#pragma unroll
                            for (int e = 0; e < width; e += 4)
                                *reinterpret_cast<f32x4*>(o + d + e) =
                                    f32x4{acc[t + e][i], acc[t + e + 1][i], acc[t + e + 2][i], acc[t + e + 3][i]} * over;
                        } else {
                            *reinterpret_cast<float2*>(o + d) = make_float2(acc[t][i] * over, acc[t + 1][i] * over);
                        }
                    });
                } else {
                    uint16_t* o = reinterpret_cast<uint16_t*>(a.out + row * a.out_stride) + at;
                    each_run([&](int t, int i, int width, int d) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < width; e += 2) w[e / 2] = T::pair(acc[t + e][i] * over, acc[t + e + 1][i] * over);
                        if (width == 8)
                            *reinterpret_cast<uint4*>(o + d) = make_uint4(w[0], w[1], w[2], w[3]);
                        else if (width == 4)
                            *reinterpret_cast<uint2*>(o + d) = make_uint2(w[0], w[1]);
                        else
                            *reinterpret_cast<uint32_t*>(o + d) = w[0];
                    });
                }
                if (a.lse && g == 0) a.lse[(int64_t)row * a.q_heads + head0 + col] = log_sum(m, l);
            } else {
                // an entry of the share: 1 for a row that starts in it, 0 for one that goes on
                const int64_t entry = ((int64_t)(2 * share_no + (share_no == first_share)) * a.q_heads + head0 + col);
                float* o = a.part_acc + entry * D;
                each_run([&](int t, int i, int width, int d) {
                    if (width >= 4) {
#pragma unroll
                        for (int e = 0; e < width; e += 4)
                            *reinterpret_cast<f32x4*>(o + d + e) =
                                f32x4{acc[t + e][i], acc[t + e + 1][i], acc[t + e + 2][i], acc[t + e + 3][i]};
                    } else {
                        *reinterpret_cast<float2*>(o + d) = make_float2(acc[t][i], acc[t + 1][i]);
                    }
                });
                if (g == 0) a.part_ml[entry] = make_float2(m, l);
            }
        }
        if (!more) {
            if (!a.by_row && unit == 0 && lane == 0)
                a.split[share_no] = cur.end > share.to && share_no == first_share ? Split{row, first_share, parts} : Split{0, 0, 0};
            return;
        }
        cur = following;
    }
}

template <int D, class T, bool F8, bool kWide, bool kWhole, bool kStream>
hipError_t launch_one(const DecodeArgs& a, hipStream_t s) {
    constexpr int W = kWhole && !(D == 256 && !F8) ? 2 * kDecodeWaves : kDecodeWaves, kSub = decode_subtiles(D, F8);
    const uint64_t units = (uint64_t)a.kv_heads * a.head_tiles;
    const uint64_t all = kWhole ? a.n_rows * units : (a.launch_shares * units + W - 1) / W, wgs = (all + 7) / 8 * 8;
    hipLaunchKernelGGL((decode_kernel<D, T, F8, kSub, W, kWide, kWhole, kStream>), dim3((unsigned)wgs), dim3(64 * W), 0, s, a.lens, a.rows,
                       a.n_rows, a.requests, a.max_len, a.window, a.shares, a.by_units.d, a.by_units.m, a.by_units.shift,
                       (uint32_t)(wgs / 8), (uint32_t)a.uncut, a);
    return hipGetLastError();
}

template <int D, class T, bool F8>
hipError_t launch_f8(const DecodeArgs& a, hipStream_t s) {
    if (a.whole) return launch_one<D, T, F8, true, true, false>(a, s);
    if constexpr (D % 64 == 0)  // decode_streams takes no others
        if (a.stream)
            return a.wide ? launch_one<D, T, F8, true, false, true>(a, s) : launch_one<D, T, F8, false, false, true>(a, s);
    return a.wide ? launch_one<D, T, F8, true, false, false>(a, s) : launch_one<D, T, F8, false, false, false>(a, s);
}

template <int D, class T>
hipError_t launch_dim(const DecodeArgs& a, bool f8, hipStream_t s) {
    return f8 ? launch_f8<D, T, true>(a, s) : launch_f8<D, T, false>(a, s);
}

template <class T>
hipError_t launch_type(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s) {
    switch (head_dim) {
    case 64: return launch_dim<64, T>(a, f8, s);
    case 96: return launch_dim<96, T>(a, f8, s);
    case 128: return launch_dim<128, T>(a, f8, s);
    case 192: return launch_dim<192, T>(a, f8, s);
    case 256: return launch_dim<256, T>(a, f8, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace attn
