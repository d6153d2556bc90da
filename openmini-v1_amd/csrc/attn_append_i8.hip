// A step's q turned, and its k turned and v quantised into the blocks of a cache of 8-bit
// integers (openmini_rope_append_i8).
//
// A block's scale is the largest of its tokens' elements over 127, so all tokens of a call that
// fall into one block (a run: slots one apart, up to the block's end) are one unit for each head.
// A workgroup takes the runs that begin in its `chunk` of tokens, which end chunk + block - 1
// tokens on at most: 64 tokens or fewer, so that one wave finds the runs by a ballot.  Then
// for each of its heads
//   its elements go to registers (k turned by sines that are made once for all heads),
//   each run's maximum meets in LDS as the bits of |x|, which order as the numbers do and put
//   NaN last,
//   every thread works out its run's scale and writes its codes; tokens that the block held
//   before are scaled again where the scale grew, by the threads of the run's tokens in turn.
// A block's old scale is read once, by the run's first lane, before the workgroup's barrier,
// and written by a thread behind it.  So no order of workgroups matters: a run has one.
//
// Growing by a quarter at least bounds what rounding again and again can add to an element
// (1/2 + 1/2 / 1.25 + ... < 2.5 steps) and leaves most blocks at one or two scales; always to
// the present maximum, a block that fills token by token would be rounded at each new
// maximum, however little above the last.
//
// q goes as in openmini_rope_apply, in the same launch, behind the workgroups of k and v.
//
// Bound by memory once the loads of the next head are on their way before a head's barrier and the
// registers of k's and v's own instances are few enough for five workgroups a CU (both in one: three).
// Measured (MI355X, one launch): 8191 tokens of 32 heads of 128, q in fp16, float in 104 us (538 MB, 5.1
// TB/s), fp16 or bf16 in 119 (336 MB, 2.8); 200 requests' tokens of 64 and 8 heads 6.3 us, one token 4.5, where no block
// grows.  Growing blocks are a thread's loop of a load, a wait and a store for each held token: one token
// behind 8, 15 and 31 held ones 7.4, 12 and 15 us; 200 requests of which a quarter of the heads' blocks grow
// 15 us in blocks of 16, 41 in blocks of 32 (all of them: 17, 43).  Prompts do not show it (103).
#include "attn_rope.hpp"

namespace attn {
namespace {

constexpr float kLeastScale = 9.094947017729282e-13f;  // 2^-40
constexpr uint32_t kMostRuns = 32;                     // tokens of a chunk
constexpr uint32_t kMostHeads = 8;                     // of a workgroup
static_assert(kMostRuns * (kMaxI8Dim / 8) <= 4 * kRopeThreads, "four items a thread hold a chunk");

struct Runs {
    int32_t of[64];     // a token's run (the lane of its first token), or -1
    int32_t token[64];  // those that have a run of the workgroup's, in order
    uint32_t tokens;    // how many
    int64_t place[64];  // byte offset of a token's slot
    int64_t scale_at[kMostRuns];
    int64_t block_at[kMostRuns];  // byte offset of the block's first token
    int32_t held[kMostRuns];      // tokens before the run's in its block
    int32_t count[kMostRuns];     // tokens of the run
    float old[kMostHeads][kMostRuns];
    uint32_t most[kMostHeads][kMostRuns];  // bits of the largest |x|
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t magnitude(float4 v) {
    return max(max(magnitude(v.x), magnitude(v.y)), max(magnitude(v.z), magnitude(v.w)));
}
// Over four neighbouring lanes, which hold items of one token and head.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));  // quad_perm 1 0 3 2
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));  // 2 3 0 1
}

__device__ __forceinline__ float new_scale(uint32_t most, int held, float old) {
    if (most >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const float need = fmaxf(__uint_as_float(most) * (1.0f / 127), kLeastScale);
    if (held == 0) return need;
    return old < need ? fmaxf(need, old * 1.25f) : old;  // a NaN stays
}

__device__ __forceinline__ uint32_t code(float x) { return (uint32_t)(int)fminf(fmaxf(rintf(x), -127.0f), 127.0f) & 255u; }
__device__ __forceinline__ uint32_t codes(float4 v, float by) {
    return code(v.x * by) | code(v.y * by) << 8 | code(v.z * by) << 16 | code(v.w * by) << 24;
}
__device__ __forceinline__ uint32_t scaled_codes(uint32_t c, float by) {
    return codes(make_float4((float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)(int8_t)(c >> 24)), by);
}

// k or v of the runs of a chunk.  Its tokens are as many as the chunk's where these follow each other
// or are all by themselves, and kItems items a thread hold them; the next head's loads are behind this
// one's barrier then.  Up to chunk + block - 1 they can be: then each head is read twice.
template <int kIn, bool kStream, int kItems, bool kValues>
__device__ __forceinline__ void kv_workgroup(AppendI8Args a, int head_dim, uint32_t chunk, uint32_t head_group) {
    extern __shared__ __attribute__((aligned(16))) float sines[];  // [tokens][pairs], and as many cosines
    __shared__ Runs runs;
    constexpr int kSize = kIn == OPENMINI_ATTN_F32 ? 4 : 2;
    RopeArgs r = a.r;
    const uint32_t tid = threadIdx.x, block = 1u << a.scales.shift, window = a.chunk + block - 1, per_head = r.per_head.d;
    const int64_t token0 = (int64_t)chunk * a.chunk;
    const int32_t head0 = (int32_t)(head_group * a.wg_heads), heads = min((int32_t)a.wg_heads, r.kv_heads - head0);
    float* scale_of = kValues ? a.scales.v : a.scales.k;
    if (tid < 64) {
        const int64_t token = token0 + tid;
        const bool mine = tid < window && token < r.tokens;
        const int32_t slot = mine ? r.slots[token] : -1;
        int32_t before = __shfl_up(slot, 1);
        if (tid == 0) before = token0 > 0 ? r.slots[token0 - 1] : -1;
        const bool real = slot >= 0 && (uint32_t)slot < r.cache.slots;
        const uint32_t at = (uint32_t)slot & (block - 1);
        const bool leads = real && (at == 0 || before != slot - 1);
        const uint64_t lead_mask = __ballot(leads), real_mask = __ballot(real);
        const uint64_t upto = lead_mask & (~0ull >> (63 - tid));
        const int32_t first = real && upto ? 63 - __clzll((long long)upto) : -1;
        const bool owned = first >= 0 && (uint32_t)first < a.chunk;
        const uint64_t owned_mask = __ballot(owned);
        int64_t place = 0;
        if (real) {
            const uint32_t page = r.cache.page.div((uint32_t)slot), in_page = (uint32_t)slot - page * r.cache.page.d;
            place = (int64_t)page * r.cache.page_stride + (int64_t)in_page * r.cache.token_stride;
            if (leads && tid < a.chunk) {
                // tokens up to the next run, the next that has no slot, or the window's end
                const uint64_t behind = tid < 63 ? (lead_mask | ~real_mask) >> (tid + 1) : 0;
                runs.count[tid] = min((int32_t)(behind ? __ffsll((unsigned long long)behind) : 64), (int32_t)(window - tid));
                runs.held[tid] = (int32_t)at;
                runs.block_at[tid] = place - (int64_t)at * r.cache.token_stride;
                const int64_t scale_at = (int64_t)page * a.scales.page_stride +
                                         (int64_t)(in_page >> a.scales.shift) * a.scales.block_stride + head0 * a.scales.head_stride;
                runs.scale_at[tid] = scale_at;
                for (int32_t h = 0; h < heads; ++h) runs.old[h][tid] = at ? scale_of[scale_at + h * a.scales.head_stride] : 0.0f;
            }
        }
        runs.of[tid] = owned ? first : -1;
        runs.place[tid] = place;
        if (owned) runs.token[__popcll(owned_mask & (((uint64_t)1 << tid) - 1))] = (int32_t)tid;
        if (tid == 0) runs.tokens = (uint32_t)__popcll(owned_mask);
    } else {
        for (uint32_t i = tid - 64; i < kMostHeads * kMostRuns; i += kRopeThreads - 64) (&runs.most[0][0])[i] = 0;
    }
    __syncthreads();
    const uint32_t tokens = runs.tokens, items = tokens * per_head;
    if (!tokens) return;

    // An item: eight elements of a token's head.
    struct Place {
        int32_t token, run, first, second, pair, u;
    };
    auto place_of = [&](uint32_t at) {
        Place p;
        const uint32_t t = r.per_head.div(at);
        p.u = (int32_t)(at - t * per_head);
        p.token = runs.token[min(t, 63u)];
        p.run = runs.of[p.token & 63];
        const bool turns = !kValues && p.u * 4 < r.n_pairs, halves = turns && !r.adjacent;
        p.pair = turns ? p.u * 4 : -1;
        p.first = halves ? p.u * 4 : p.u * 8;
        p.second = halves ? p.u * 4 + r.n_pairs : p.u * 8 + 4;
        return p;
    };
    const int64_t stride = kValues ? r.v_stride : r.k_stride;
    const uint8_t* src = (kValues ? r.v : r.k) + token0 * stride + (int64_t)head0 * head_dim * kSize;
    uint8_t* cache = (kValues ? r.cache.v : r.cache.k) + (int64_t)head0 * r.cache.head_stride;
    auto load_item = [&](const Place& p, int32_t h, float4* x, float4* y) {
        const uint8_t* from = src + p.token * stride + (int64_t)h * head_dim * kSize;
        *x = load4<kIn, kStream>(from + p.first * kSize);
        *y = load4<kIn, kStream>(from + p.second * kSize);
    };
    const float* cosines = sines + window * r.n_pairs;
    auto turned = [&](const Place& p, float4& x, float4& y) {
        if constexpr (!kValues)
            if (p.pair >= 0) {
                const uint32_t at = (uint32_t)p.token * (uint32_t)r.n_pairs + (uint32_t)p.pair;
                turn(x, y, *reinterpret_cast<const float4*>(sines + at), *reinterpret_cast<const float4*>(cosines + at), r.adjacent);
            }
    };
    auto tell = [&](const Place& p, int32_t h, bool real, float4 x, float4 y) {  // its run's maximum
        uint32_t most = real ? max(magnitude(x), magnitude(y)) : 0;
        if (per_head % 4 == 0) most = quad_max(most);
        if (real && (per_head % 4 || (tid & 3) == 0)) atomicMax(&runs.most[h][p.run], most);
    };
    auto write = [&](const Place& p, int32_t h, float4 x, float4 y) {
        const int32_t held = runs.held[p.run];
        const float old = runs.old[h][p.run], scale = new_scale(runs.most[h][p.run], held, old);
        const float by = scale == scale ? 1.0f / scale : 0.0f;
        uint8_t* to = cache + h * r.cache.head_stride;
        uint8_t* c = to + runs.place[p.token];
        const u32x2 w = {codes(x, by), codes(y, by)};
        if (p.second == p.first + 4) {
            *reinterpret_cast<u32x2*>(c + p.first) = w;
        } else {
            *reinterpret_cast<uint32_t*>(c + p.first) = w[0];
            *reinterpret_cast<uint32_t*>(c + p.second) = w[1];
        }
        const int32_t nth = p.token - p.run;
        if (p.u == 0 && nth == 0) scale_of[runs.scale_at[p.run] + h * a.scales.head_stride] = scale;
        if (held && scale > old) {  // not where either is NaN
            const float again = old / scale;
            for (int32_t t = nth; t < held; t += runs.count[p.run]) {
                u32x2* was = reinterpret_cast<u32x2*>(to + runs.block_at[p.run] + t * r.cache.token_stride + p.u * 8);
                const u32x2 v = *was;
                *was = u32x2{scaled_codes(v[0], again), scaled_codes(v[1], again)};
            }
        }
    };
    const bool once = items <= kItems * kRopeThreads;
    Place at[kItems];
    float4 lo[kItems], hi[kItems];
    if (once)
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            at[i] = place_of(tid + i * kRopeThreads);
            if (tid + i * kRopeThreads < items) load_item(at[i], 0, &lo[i], &hi[i]);
        }
    if constexpr (!kValues) {
        for (uint32_t j = tid; j < tokens * (uint32_t)r.n_pairs; j += kRopeThreads) {
            const uint32_t t = r.by_pairs.div(j), i = j - t * r.by_pairs.d, token = (uint32_t)runs.token[t];
            const RopePair pair = r.pairs[i];
            const int32_t p = r.positions[pair.axis * r.position_stride + token0 + token];
            float s, c;
            sin_cos((uint64_t)(int64_t)p * pair.step, &s, &c);
            sines[token * r.n_pairs + i] = s * r.scale;
            sines[(window + token) * r.n_pairs + i] = c * r.scale;
        }
        __syncthreads();
    }
    if (!once) {
        for (int32_t h = 0; h < heads; ++h) {
            for (int pass = 0; pass < 2; ++pass) {
                for (uint32_t n = tid; n < (items + 63) / 64 * 64; n += kRopeThreads) {
                    const Place p = place_of(min(n, items - 1));
                    float4 x, y;
                    load_item(p, h, &x, &y);
                    turned(p, x, y);
                    if (pass == 0)
                        tell(p, h, n < items, x, y);
                    else if (n < items)
                        write(p, h, x, y);
                }
                __syncthreads();
            }
        }
        return;
    }
    for (int32_t h = 0; h < heads; ++h) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const bool real = tid + i * kRopeThreads < items;
            if (real) turned(at[i], lo[i], hi[i]);
            tell(at[i], h, real, lo[i], hi[i]);
        }
        float4 x[kItems], y[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            x[i] = lo[i];
            y[i] = hi[i];
            if (h + 1 < heads && tid + i * kRopeThreads < items) load_item(at[i], h + 1, &lo[i], &hi[i]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kItems; ++i)
            if (tid + i * kRopeThreads < items) write(at[i], h, x[i], y[i]);
    }
}

template <int kIn, bool kStream, int kTokens, int kItems>
__global__ __launch_bounds__(kRopeThreads) void append_i8_kernel(AppendI8Args a, int head_dim, uint32_t beside) {
    if (blockIdx.x < a.kv_wgs) {
        const uint32_t part = blockIdx.x >> 1, chunk = a.by_head_groups.div(part);
        if (blockIdx.x & 1)
            kv_workgroup<kIn, kStream, kItems, true>(a, head_dim, chunk, part - chunk * a.by_head_groups.d);
        else
            kv_workgroup<kIn, kStream, kItems, false>(a, head_dim, chunk, part - chunk * a.by_head_groups.d);
    } else {
        const uint32_t at = blockIdx.x - a.kv_wgs, group = a.by_slices.div(at);
        rope_workgroup<kIn, kStream, kTokens>(a.r, head_dim, beside, group, at - group * a.by_slices.d);
    }
}

template <int kIn, int kItems>
hipError_t launch_items(const AppendI8Args& a, int head_dim, uint32_t beside, bool stream, uint32_t wgs, size_t lds, hipStream_t s) {
    if (stream)
        hipLaunchKernelGGL((append_i8_kernel<kIn, true, batch_of(kIn), kItems>), dim3(wgs), dim3(kRopeThreads), lds, s, a, head_dim, beside);
    else
        hipLaunchKernelGGL((append_i8_kernel<kIn, false, 1, kItems>), dim3(wgs), dim3(kRopeThreads), lds, s, a, head_dim, beside);
    return hipGetLastError();
}

template <int kIn>
hipError_t launch_type(const AppendI8Args& a, int head_dim, uint32_t beside, bool stream, uint32_t wgs, size_t lds, hipStream_t s) {
    const uint32_t items = a.chunk * a.r.per_head.d;
    if (items <= kRopeThreads) return launch_items<kIn, 1>(a, head_dim, beside, stream, wgs, lds, s);
    if (items <= 2 * kRopeThreads) return launch_items<kIn, 2>(a, head_dim, beside, stream, wgs, lds, s);
    return launch_items<kIn, 4>(a, head_dim, beside, stream, wgs, lds, s);
}

}  // namespace

hipError_t launch_append_i8(AppendI8Args& a, int head_dim, hipStream_t s) {
    RopeArgs& r = a.r;
    const uint32_t items = r.per_token.d, slices = (items + kRopeThreads - 1) / kRopeThreads;
    uint32_t beside = 1;
    if (items < kRopeThreads) beside = kRopeThreads / items < kMostBeside ? kRopeThreads / items : kMostBeside;
    const uint32_t block = 1u << a.scales.shift;
    a.chunk = block > 16 ? block : 16;
    const uint32_t chunks = (uint32_t)(((int64_t)r.tokens + a.chunk - 1) / a.chunk);
    const bool stream = ((int64_t)r.tokens + beside - 1) / beside * slices > 2048;
    a.wg_heads = 1;
    while (a.wg_heads < kMostHeads && (int64_t)chunks * r.kv_heads > (int64_t)a.wg_heads * 2048) a.wg_heads *= 2;
    a.by_head_groups = FastDiv(((uint32_t)r.kv_heads + a.wg_heads - 1) / a.wg_heads);
    a.by_slices = FastDiv(slices);
    a.kv_wgs = 2 * chunks * a.by_head_groups.d;
    const int64_t batch = stream ? (int64_t)batch_of(r.x_dtype) * beside : beside;
    a.q_groups = (uint32_t)((r.tokens + batch - 1) / batch);
    const uint32_t wgs = a.kv_wgs + a.q_groups * slices;
    const size_t q_lds = 2 * 4 * (size_t)batch * r.n_pairs, kv_lds = 2 * 4 * (size_t)(a.chunk + block - 1) * r.n_pairs;
    const size_t lds = q_lds > kv_lds ? q_lds : kv_lds;
    if (r.x_dtype == OPENMINI_ATTN_F32) return launch_type<OPENMINI_ATTN_F32>(a, head_dim, beside, stream, wgs, lds, s);
    if (r.x_dtype == OPENMINI_ATTN_F16) return launch_type<OPENMINI_ATTN_F16>(a, head_dim, beside, stream, wgs, lds, s);
    return launch_type<OPENMINI_ATTN_BF16>(a, head_dim, beside, stream, wgs, lds, s);
}

}  // namespace attn
