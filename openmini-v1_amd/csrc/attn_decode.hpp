// Attention of single query tokens over a paged cache (openmini_attn_decode).
//
// A row's query heads that share a key head are the columns of 16 x 16 MFMA tiles.  A wave
// takes 32 keys at a time:
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
// The probabilities enter the second product as the sum of two 16-bit parts (their rounding
// to one would be 2^-9 of the output in bf16; the second product is a tenth of the time that
// its keys take to arrive).  Sums, maxima and the joined parts are fp32.
//
// Bound by memory: 4 operations a byte and key head's query head.  The loads of the next
// keys are issued as soon as the registers of the present ones are free, so a wave has one
// tile in flight all the time and the waves of a CU together some 100 KB, several times
// what latency times bandwidth asks for.
#pragma once

#include <type_traits>

#include "attn_internal.hpp"
#include "qmm_device.hpp"

namespace attn {

using qmm::bf16x8;
using qmm::f16x8;
using qmm::f32x4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct BF16 {
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

template <int kBytes>
__device__ __forceinline__ void load(const uint8_t* p, uint32_t* d) {
    if constexpr (kBytes == 16) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = v[i];
    } else if constexpr (kBytes == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        d[0] = v.x;
        d[1] = v.y;
    } else if constexpr (kBytes == 4) {
        d[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        d[0] = *reinterpret_cast<const uint16_t*>(p);
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

// The part of a row that a workgroup takes: tiles [tile0, tile1) of keys [lo, hi), part
// `part` of `parts`, whose first sits at `place` among the parts of all split rows.
struct Part {
    uint32_t row, tile0, tile1, part, parts, place;
    int32_t lo, hi;
};

struct Span {
    int32_t lo, hi;
    uint32_t tiles;
};

// The keys that row r sees: none for a request outside the tables.
__device__ __forceinline__ Span span_of(const DecodeArgs& a, uint32_t r) {
    Span s;
    s.hi = min(max(a.lens[r], 0), (int32_t)a.max_len);
    const uint32_t request = a.rows ? (uint32_t)a.rows[r] : r;
    if (request >= a.requests) s.hi = 0;
    s.lo = a.window && (int64_t)s.hi > a.window ? s.hi - (int32_t)a.window : 0;
    s.tiles = (uint32_t)((s.hi + kTile - 1) / kTile - s.lo / kTile);  // max_len leaves room for + 31
    return s;
}

__device__ __forceinline__ uint32_t parts_of(const Span& s, uint32_t part_tiles) {
    return min(max((s.tiles + part_tiles - 1) / part_tiles, 1u), (uint32_t)kMaxParts);
}

__device__ __forceinline__ void fill(Part& p, uint32_t row, const Span& s, uint32_t parts, uint32_t part, uint32_t place) {
    const uint32_t base = (uint32_t)(s.lo / kTile);
    p.row = row;
    p.lo = s.lo;
    p.hi = s.hi;
    p.parts = parts;
    p.part = part;
    p.place = place;
    // tiles spread evenly: part i has (i + 1) n / parts - i n / parts of them
    p.tile0 = base + (uint32_t)((uint64_t)part * s.tiles / parts);
    p.tile1 = base + (uint32_t)((uint64_t)(part + 1) * s.tiles / parts);
}

// The item-th part of the call, or false.  A part has about total / target_parts tiles: the
// lengths of the call alone decide, so long rows beside short ones are cut into as many
// parts as their share of the work.
template <int W>
__device__ __forceinline__ bool find_part(const DecodeArgs& a, uint32_t item, Part& out) {
    const uint32_t lane = threadIdx.x & 63;
    if (a.n_rows <= 64) {  // every wave by itself
        Span s = {0, 0, 0};
        if (lane < a.n_rows) s = span_of(a, lane);
        const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)wave_sums(s.tiles), 63);
        const uint32_t part_tiles = max(a.min_tiles, (total + a.target_parts - 1) / a.target_parts);
        const uint32_t n = lane < a.n_rows ? parts_of(s, part_tiles) : 0;
        const uint32_t upto = wave_sums(n), places = wave_sums(n > 1 ? n : 0);
        const uint64_t hit = __ballot(item >= upto - n && item < upto);
        if (!hit) return false;
        const int at = __ffsll((unsigned long long)hit) - 1;
        s.lo = __builtin_amdgcn_readlane(s.lo, at);
        s.hi = __builtin_amdgcn_readlane(s.hi, at);
        s.tiles = (uint32_t)__builtin_amdgcn_readlane((int)s.tiles, at);
        const uint32_t parts = (uint32_t)__builtin_amdgcn_readlane((int)n, at);
        fill(out, (uint32_t)at, s, parts, item - ((uint32_t)__builtin_amdgcn_readlane((int)upto, at) - parts),
             (uint32_t)__builtin_amdgcn_readlane((int)places, at) - (parts > 1 ? parts : 0));
        return true;
    }
    __shared__ uint32_t wave_total[2][W], found[7];
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t each = (a.n_rows + 64 * W - 1) / (64 * W);
    const uint32_t r0 = min(threadIdx.x * each, a.n_rows), r1 = min(r0 + each, a.n_rows);
    uint32_t v = 0;
    for (uint32_t r = r0; r < r1; ++r) v += span_of(a, r).tiles;
    uint32_t sum = wave_sums(v);
    if (lane == 63) wave_total[0][wave] = sum;
    if (threadIdx.x == 0) found[0] = 0xFFFFFFFFu;
    __syncthreads();
    uint32_t total = 0;
    for (int w = 0; w < W; ++w) total += wave_total[0][w];
    const uint32_t part_tiles = max(a.min_tiles, (total + a.target_parts - 1) / a.target_parts);
    uint32_t n = 0, split = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const uint32_t p = parts_of(span_of(a, r), part_tiles);
        n += p;
        split += p > 1 ? p : 0;
    }
    uint32_t upto = wave_sums(n), places = wave_sums(split);
    __syncthreads();
    if (lane == 63) {
        wave_total[0][wave] = upto;
        wave_total[1][wave] = places;
    }
    __syncthreads();
    upto -= n;
    places -= split;
    for (uint32_t w = 0; w < wave; ++w) {
        upto += wave_total[0][w];
        places += wave_total[1][w];
    }
    if (item >= upto && item < upto + n) {
        for (uint32_t r = r0; r < r1; ++r) {
            const Span s = span_of(a, r);
            const uint32_t p = parts_of(s, part_tiles);
            if (item < upto + p) {
                found[0] = r;
                found[1] = p;
                found[2] = item - upto;
                found[3] = places;
                found[4] = (uint32_t)s.lo;
                found[5] = (uint32_t)s.hi;
                found[6] = s.tiles;
                break;
            }
            upto += p;
            places += p > 1 ? p : 0;
        }
    }
    __syncthreads();
    if (found[0] == 0xFFFFFFFFu) return false;
    Span s;
    s.lo = (int32_t)found[4];
    s.hi = (int32_t)found[5];
    s.tiles = found[6];
    fill(out, found[0], s, found[1], found[2], found[3]);
    return true;
}

template <int D, class T, bool F8, int W>
__global__ __launch_bounds__(64 * W) void decode_kernel(DecodeArgs a) {
    constexpr int kEl = F8 ? 1 : 2;           // bytes of a cache element
    constexpr int kSteps = D / 32;            // MFMAs over head_dim of the first product
    constexpr int kTiles = D / 16;            // 16-dimension tiles of the second
    constexpr int kKWords = kSteps * 2 * kEl; // dwords of a key in a lane
    constexpr int kVWords = (kTiles * kEl + 3) / 4;
    // V in chunks of 128, 64 and 32 dimensions, of which a lane holds 8, 4 and 2
    constexpr int kFull = D / 128, kRest = D % 128;
    constexpr bool kHas64 = kRest >= 64, kHas32 = kRest % 64 != 0;
    constexpr int kRow = D + 4;  // LDS row of a head: neighbours start four banks apart

    // Two uses, one after the other: accumulators of half the waves; weights of a row's
    // parts and the sums of their groups.
    constexpr int kRed = W / 2 * kHeadTile * kRow;
    constexpr int kJoin = kMaxParts * kHeadTile + 64 * W * 4;
    __shared__ __attribute__((aligned(16))) float red[kRed > kJoin ? kRed : kJoin];
    __shared__ float wave_m[W][kHeadTile], wave_l[W][kHeadTile], all_m[kHeadTile], all_l[kHeadTile];
    __shared__ uint32_t is_last;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int col = lane & 15, g = lane >> 4;

    // Workgroups go round the 8 XCDs by index; those of one key head's head tiles read the
    // same keys and take the same XCD, whose L2 then reads them once.
    const uint32_t y = blockIdx.x >> 3;
    const uint32_t head_tile = y - a.by_head_tiles.div(y) * a.by_head_tiles.d;
    const uint32_t pos = a.by_head_tiles.div(y) * 8 + (blockIdx.x & 7);
    const uint32_t item = a.by_kv_heads.div(pos), kv = pos - item * a.by_kv_heads.d;
    Part part;
    if (!find_part<W>(a, item, part)) return;
    const int heads = min(kHeadTile, a.group - (int)head_tile * kHeadTile);  // columns in use
    const int head0 = (int)kv * a.group + (int)head_tile * kHeadTile;

    // q^T: lane holds column `col`, eight dimensions a step, in the order of a key's loads
    u32x4 qf[kSteps];
    {
        const uint8_t* q = a.q + part.row * a.q_stride + (int64_t)(head0 + min(col, heads - 1)) * D * 2;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const int dim = F8 && (st | 1) < kSteps ? (st >> 1) * 64 + g * 16 + (st & 1) * 8 : st * 32 + g * 8;
            qf[st] = *reinterpret_cast<const u32x4*>(q + dim * 2);
            if (col >= heads) qf[st] = u32x4{0, 0, 0, 0};
        }
    }

    f32x4 acc[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0;

    const uint32_t request = a.rows ? (uint32_t)a.rows[part.row] : part.row;
    const int32_t* table = a.tables + (int64_t)request * a.table_stride;
    const int32_t first_group = part.lo & ~7, last_group = (part.hi - 1) & ~7;
    const uint8_t* k_lane = a.cache.k + kv * a.cache.head_stride + g * 16;
    const uint8_t* v_base = a.cache.v + kv * a.cache.head_stride;
    const int kg = col >> 2, k_row = col & 3;  // the lane's key of tile s: 8 kg + 4 s + k_row

    // the eight keys from 8 * grp of a tile on: their page's column, kept inside [lo, hi)
    auto group_at = [&](uint32_t tile, int grp) -> int32_t {
        return min(max((int32_t)(tile * kTile) + 8 * grp, first_group), last_group);
    };
    auto page_at = [&](int32_t key) -> int32_t { return table[a.cache.page.div((uint32_t)key)]; };
    auto offset_of = [&](int32_t page, int32_t key) -> int64_t {
        const uint32_t in_page = (uint32_t)key - a.cache.page.div((uint32_t)key) * a.cache.page.d;
        return ((uint32_t)page < a.cache.n_pages ? (int64_t)page * a.cache.page_stride : 0) +
               (int64_t)in_page * a.cache.token_stride;
    };

    uint32_t kraw[2][kKWords], vraw[8][kVWords];
    auto load_k = [&](uint32_t tile, int32_t page) {
        const uint8_t* p = k_lane + offset_of(page, group_at(tile, kg)) + k_row * a.cache.token_stride;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint8_t* ps = p + 4 * s * a.cache.token_stride;
            if constexpr (F8) {
#pragma unroll
                for (int c = 0; c < kSteps / 2; ++c) load<16>(ps + c * 64, &kraw[s][4 * c]);
                if constexpr (kSteps & 1) load<8>(ps - g * 8 + (kSteps - 1) * 32, &kraw[s][2 * (kSteps - 1)]);
            } else {
#pragma unroll
                for (int st = 0; st < kSteps; ++st) load<16>(ps + st * 64, &kraw[s][4 * st]);
            }
        }
    };
    auto load_v = [&](uint32_t tile, int32_t page) {
        const uint8_t* p = v_base + offset_of(page, group_at(tile, g));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t* pj = p + j * a.cache.token_stride;
#pragma unroll
            for (int c = 0; c < kFull; ++c) load<8 * kEl>(pj + (c * 128 + col * 8) * kEl, &vraw[j][c * 2 * kEl]);
            if constexpr (kHas64) load<4 * kEl>(pj + (kFull * 128 + col * 4) * kEl, &vraw[j][kFull * 2 * kEl]);
            if constexpr (kHas32)
                load<2 * kEl>(pj + (kFull * 128 + kHas64 * 64 + col * 2) * kEl, &vraw[j][kFull * 2 * kEl + kHas64 * kEl]);
        }
    };

    uint32_t tile = part.tile0 + wave;
    if (tile < part.tile1) {
        int32_t k_page = page_at(group_at(tile, kg)), v_page = page_at(group_at(tile, g));
        uint32_t next = min(tile + W, part.tile1 - 1);
        int32_t k_next = page_at(group_at(next, kg)), v_next = page_at(group_at(next, g));
        load_k(tile, k_page);
        load_v(tile, v_page);
        for (;;) {
            const bool more = tile + W < part.tile1;
            // first product
            f32x4 sc[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                    u32x4 kf;
                    if constexpr (F8) {
                        const uint32_t w0 = kraw[s][2 * st], w1 = kraw[s][2 * st + 1];
                        kf = u32x4{T::template from_f8<false>(w0), T::template from_f8<true>(w0),
                                   T::template from_f8<false>(w1), T::template from_f8<true>(w1)};
                    } else {
                        kf = u32x4{kraw[s][4 * st], kraw[s][4 * st + 1], kraw[s][4 * st + 2], kraw[s][4 * st + 3]};
                    }
                    sc[s] = T::mfma(kf, qf[st], sc[s]);
                }
            // the pages of the tile after the next, then the next keys: their pages came
            // with loads that have been waited for
            int32_t k_after = 0, v_after = 0;
            if (more) {
                const uint32_t after = min(tile + 2 * W, part.tile1 - 1);
                k_after = page_at(group_at(after, kg));
                v_after = page_at(group_at(after, g));
                load_k(tile + W, k_next);
            }

            float x[8];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * s + i] = sc[s][i] * a.scale;
            // keys outside the row's or on no page of the cache: only a row's first and
            // last tiles, and broken tables, have them
            const int32_t key0 = (int32_t)(tile * kTile) + 8 * g;
            const bool on_page = (uint32_t)v_page < a.cache.n_pages;
            const bool whole = on_page && key0 >= part.lo && key0 + 8 <= part.hi;
            if (!__all(whole)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool seen = on_page && key0 + j >= part.lo && key0 + j < part.hi;
                    x[j] = seen ? x[j] : -INFINITY;
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) vraw[j][w] = seen ? vraw[j][w] : 0;  // 0 * NaN is NaN
                }
            }
            const float top = column_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                               fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))));
            if (__any(top > m)) {
                const float to = fmaxf(m, top);
                const float by = exp2_of(m - above(to));
                m = to;
                l *= by;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) acc[i] *= by;
            }
            const float base = above(m);
            u32x4 p_high, p_low;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float p0 = exp2_of(x[j] - base), p1 = exp2_of(x[j + 1] - base);
                l += p0 + p1;
                const uint32_t h = T::pair(p0, p1);
                p_high[j / 2] = h;
                p_low[j / 2] = T::pair(p0 - T::low(h), p1 - T::high(h));
            }
            // second product
            auto add = [&](int t, u32x4 vf) {
                acc[t] = T::mfma(vf, p_high, acc[t]);
                acc[t] = T::mfma(vf, p_low, acc[t]);
            };
            auto chunk = [&](int tile0, int word0, auto width_tag) {
                constexpr int kWidth = decltype(width_tag)::value;
                if constexpr (F8) {
#pragma unroll
                    for (int w = 0; w < (kWidth + 3) / 4; ++w) {
                        u32x4 f[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            const uint32_t v0 = vraw[2 * p][word0 + w], v1 = vraw[2 * p + 1][word0 + w];
                            const uint32_t lo = __builtin_amdgcn_perm(v1, v0, 0x05010400u);
                            f[0][p] = T::template from_f8<false>(lo);
                            f[1][p] = T::template from_f8<true>(lo);
                            if constexpr (kWidth >= 4) {
                                const uint32_t hi = __builtin_amdgcn_perm(v1, v0, 0x07030602u);
                                f[2][p] = T::template from_f8<false>(hi);
                                f[3][p] = T::template from_f8<true>(hi);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < (kWidth < 4 ? kWidth : 4); ++e) add(tile0 + 4 * w + e, f[e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < kWidth; ++e) {
                        u32x4 f;
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            f[p] = __builtin_amdgcn_perm(vraw[2 * p + 1][word0 + e / 2], vraw[2 * p][word0 + e / 2],
                                                         e & 1 ? 0x07060302u : 0x05040100u);
                        add(tile0 + e, f);
                    }
                }
            };
#pragma unroll
            for (int c = 0; c < kFull; ++c) chunk(8 * c, c * 2 * kEl, std::integral_constant<int, 8>{});
            if constexpr (kHas64) chunk(8 * kFull, kFull * 2 * kEl, std::integral_constant<int, 4>{});
            if constexpr (kHas32)
                chunk(8 * kFull + 4 * kHas64, kFull * 2 * kEl + kHas64 * kEl, std::integral_constant<int, 2>{});
            if (!more) break;
            load_v(tile + W, v_next);
            tile += W;
            v_page = v_next;
            k_next = k_after;
            v_next = v_after;
        }
    }

    // The waves' sums joined: to a common maximum, then the upper half's accumulators into
    // the lower half's, then the lower half's over all threads.
    l = column_sum(l);
    if (g == 0) {
        wave_m[wave][col] = m;
        wave_l[wave][col] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, wave_m[w][col]);
    const float base = above(top);
#pragma unroll
    for (int w = 0; w < W; ++w) sum += exp2_of(wave_m[w][col] - base) * wave_l[w][col];
    const float by = exp2_of(m - base);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i] *= by;
    if (wave == 0 && g == 0) {
        all_m[col] = top;
        all_l[col] = sum;
    }
    // accumulator i of tile t is dimension chunk + (4 g + i) * width + (t in the chunk)
    auto each_acc = [&](auto&& f) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int c = t / 8 < kFull ? t / 8 * 8 : kHas64 && t < 8 * kFull + 4 ? 8 * kFull : 8 * kFull + 4 * kHas64;
            const int width = t / 8 < kFull ? 8 : kHas64 && t < 8 * kFull + 4 ? 4 : 2;
#pragma unroll
            for (int i = 0; i < 4; ++i) f(t, i, c * 16 + (4 * g + i) * width + (t - c));
        }
    };
    float* mine = red + ((wave % (W / 2)) * kHeadTile + col) * kRow;
    if (wave >= W / 2 && col < heads) each_acc([&](int t, int i, int d) { mine[d] = acc[t][i]; });
    __syncthreads();
    if (wave < W / 2 && col < heads) each_acc([&](int t, int i, int d) { mine[d] += acc[t][i]; });
    __syncthreads();

    const int outs = heads * (D / 4);  // fours of the output
    const uint32_t units = (uint32_t)(a.kv_heads * a.head_tiles), unit = kv * a.head_tiles + head_tile;
    auto store = [&](int o, f32x4 v, float total) {
        const int h = o / (D / 4), d = o % (D / 4) * 4;
        const float over = total > 0 || total != total ? a.cache.v_scale / total : 0.0f;
        v *= over;
        const int64_t at = (int64_t)(head0 + h) * D + d;
        if (a.out_f32)
            *reinterpret_cast<f32x4*>(a.out + part.row * a.out_stride + at * 4) = v;
        else
            *reinterpret_cast<uint2*>(a.out + part.row * a.out_stride + at * 2) =
                make_uint2(T::pair(v[0], v[1]), T::pair(v[2], v[3]));
    };
    auto store_lse = [&](int h, float most, float total) {
        if (a.lse)
            a.lse[(int64_t)part.row * a.q_heads + head0 + h] =
                total == 0 ? -INFINITY : (most + __builtin_amdgcn_logf(total)) * 0.693147180559945309f;
    };
    auto waves_sum = [&](int o) {
        const float* r = red + o / (D / 4) * kRow + o % (D / 4) * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(r);
#pragma unroll
        for (int w = 1; w < W / 2; ++w) v += *reinterpret_cast<const f32x4*>(r + w * kHeadTile * kRow);
        return v;
    };
    if (part.parts == 1) {
        for (int o = tid; o < outs; o += 64 * W) store(o, waves_sum(o), all_l[o / (D / 4)]);
        if (tid < heads) store_lse(tid, all_m[tid], all_l[tid]);
        return;
    }

    // A part of a split row: its sums to the workspace, past this XCD's L2 (sc1), and the
    // last of the row's workgroups adds the parts.  As in the batched GEMV's K split: each
    // wave's stores are acknowledged (vmcnt 0) before the barrier that precedes the count,
    // the loads follow the count's return and miss this XCD's L2 (sc1); no workgroup waits
    // for another.
    constexpr int kSc1 = 16;
    const __amdgpu_buffer_rsrc_t acc_rsrc = qmm::make_rsrc(a.part_acc, a.part_acc_bytes);
    const __amdgpu_buffer_rsrc_t ml_rsrc = qmm::make_rsrc(a.part_ml, a.part_ml_bytes);
    const int tile_heads = min(kHeadTile, a.group);  // heads of a workspace entry
    auto entry = [&](uint32_t i) { return ((part.place + i) * units + unit) * (uint32_t)tile_heads; };
    for (int o = tid; o < outs; o += 64 * W)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, waves_sum(o)), acc_rsrc,
                                               (int)(entry(part.part) * (D * 4) + o * 16), 0, kSc1);
    if (tid < heads) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(all_m[tid]), __float_as_uint(all_l[tid])}, ml_rsrc,
                                              (int)((entry(part.part) + tid) * 8), 0, kSc1);
    }
    __builtin_amdgcn_s_waitcnt(qmm::vmcnt_only(0));
    __syncthreads();
    if (tid == 0) {
        uint32_t* count = a.counters + (size_t)part.place * units + unit;
        const bool last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == part.parts - 1;
        if (last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        is_last = last;
    }
    __syncthreads();
    if (!is_last) return;

    // weight of part i for each head, in `red`
    for (int h = wave; h < heads; h += W) {
        float pm[kMaxParts / 64], pl[kMaxParts / 64], most = -INFINITY, total = 0;
#pragma unroll
        for (int c = 0; c < kMaxParts / 64; ++c) {
            const uint32_t i = c * 64 + lane;
            pm[c] = -INFINITY;
            pl[c] = 0;
            if (i < part.parts) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(ml_rsrc, (int)((entry(i) + h) * 8), 0, kSc1);
                pm[c] = __uint_as_float(v[0]);
                pl[c] = __uint_as_float(v[1]);
            }
            most = fmaxf(most, pm[c]);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
#pragma unroll
        for (int c = 0; c < kMaxParts / 64; ++c) {
            const uint32_t i = c * 64 + lane;
            const float w = exp2_of(pm[c] - above(most));
            if (i < part.parts) red[i * kHeadTile + h] = w;
            total += w * pl[c];
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
        if (lane == 0) {
            all_m[h] = most;
            all_l[h] = total;
        }
    }
    __syncthreads();
    // groups of threads take every groups-th part; their sums are added in order
    const int groups = max(64 * W / outs, 1);
    f32x4* sums = reinterpret_cast<f32x4*>(red + kMaxParts * kHeadTile);
    for (int o0 = 0; o0 < outs; o0 += 64 * W) {
        const int grp = groups == 1 ? 0 : tid / outs, o = groups == 1 ? o0 + tid : tid % outs;
        const bool active = grp < groups && o < outs;
        f32x4 v = {0, 0, 0, 0};
        if (active) {
            const int h = o / (D / 4);
#pragma unroll 8
            for (uint32_t i = grp; i < part.parts; i += groups) {
                const u32x4 r = __builtin_amdgcn_raw_buffer_load_b128(acc_rsrc, (int)(entry(i) * (D * 4) + o * 16), 0, kSc1);
                v += __builtin_bit_cast(f32x4, r) * red[i * kHeadTile + h];
            }
        }
        if (groups > 1) {
            if (active) sums[tid] = v;
            __syncthreads();
            if (active && grp == 0)
                for (int k = 1; k < groups; ++k) v += sums[k * outs + o];
        }
        if (active && grp == 0) store(o, v, all_l[o / (D / 4)]);
    }
    if (tid < heads) store_lse(tid, all_m[tid], all_l[tid]);
}

// Waves of a workgroup: eight where their registers let a CU hold two workgroups.
template <int D>
constexpr int decode_waves() { return D <= 128 ? 8 : 4; }

template <int D, class T, bool F8>
hipError_t launch_one(const DecodeArgs& a, hipStream_t s) {
    constexpr int W = decode_waves<D>();
    const uint64_t heads = (uint64_t)a.max_parts * a.kv_heads;
    const uint64_t wgs = (heads + 7) / 8 * 8 * a.head_tiles;
    hipLaunchKernelGGL((decode_kernel<D, T, F8, W>), dim3((unsigned)wgs), dim3(64 * W), 0, s, a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_type(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s) {
    switch (head_dim) {
    case 64: return f8 ? launch_one<64, T, true>(a, s) : launch_one<64, T, false>(a, s);
    case 96: return f8 ? launch_one<96, T, true>(a, s) : launch_one<96, T, false>(a, s);
    case 128: return f8 ? launch_one<128, T, true>(a, s) : launch_one<128, T, false>(a, s);
    case 192: return f8 ? launch_one<192, T, true>(a, s) : launch_one<192, T, false>(a, s);
    case 256: return f8 ? launch_one<256, T, true>(a, s) : launch_one<256, T, false>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace attn
