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
#include "attn_rope.hpp"

namespace attn {
namespace {

constexpr float kLeastScale = 9.094947017729282e-13f;  // 2^-40
constexpr uint32_t kMostRuns = 32;                     // tokens of a chunk
constexpr uint32_t kMostHeads = 8;                     // of a workgroup
static_assert((2 * kMostRuns - 1) * (kMaxI8Dim / 8) <= 8 * kRopeThreads, "eight items a thread hold the longest runs");

struct Runs {
    int32_t of[64];            // a token's run (the lane of its first token), or -1
    int64_t place[64];         // byte offset of its slot
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

// k or v of the runs of a chunk.  kItems: items of a thread, at most.
template <int kIn, bool kStream, int kItems>
__device__ __forceinline__ void kv_workgroup(AppendI8Args a, int head_dim, uint32_t chunk, uint32_t head_group, bool values) {
    extern __shared__ __attribute__((aligned(16))) float sines[];  // [tokens][pairs], and as many cosines
    __shared__ Runs runs;
    constexpr int kSize = kIn == OPENMINI_ATTN_F32 ? 4 : 2;
    RopeArgs r = a.r;
    const uint32_t tid = threadIdx.x, block = 1u << a.scales.shift, tokens = a.chunk + block - 1, per_head = r.per_head.d;
    const int64_t token0 = (int64_t)chunk * a.chunk;
    const int32_t head0 = (int32_t)(head_group * a.wg_heads), heads = min((int32_t)a.wg_heads, r.kv_heads - head0);
    float* scale_of = values ? a.scales.v : a.scales.k;
    if (tid < 64) {
        const int64_t token = token0 + tid;
        const bool mine = tid < tokens && token < r.tokens;
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
        int64_t place = 0;
        if (real) {
            const uint32_t page = r.cache.page.div((uint32_t)slot), in_page = (uint32_t)slot - page * r.cache.page.d;
            place = (int64_t)page * r.cache.page_stride + (int64_t)in_page * r.cache.token_stride;
            if (leads && tid < a.chunk) {
                // tokens up to the next run, the next that has no slot, or the window's end
                const uint64_t behind = tid < 63 ? (lead_mask | ~real_mask) >> (tid + 1) : 0;
                runs.count[tid] = min((int32_t)(behind ? __ffsll((unsigned long long)behind) : 64), (int32_t)(tokens - tid));
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
    } else {
        for (uint32_t i = tid - 64; i < kMostHeads * kMostRuns; i += kRopeThreads - 64) (&runs.most[0][0])[i] = 0;
    }
    __syncthreads();
    float* cosines = sines + tokens * r.n_pairs;
    if (!values)
        for (uint32_t j = tid; j < tokens * (uint32_t)r.n_pairs; j += kRopeThreads) {
            const uint32_t token = r.by_pairs.div(j), i = j - token * r.by_pairs.d;
            if (runs.of[token] < 0) continue;
            const RopePair pair = r.pairs[i];
            const int32_t p = r.positions[pair.axis * r.position_stride + token0 + token];
            float s, c;
            sin_cos((uint64_t)(int64_t)p * pair.step, &s, &c);
            sines[j] = s * r.scale;
            cosines[j] = c * r.scale;
        }
    if (!values) __syncthreads();

    // the thread's items: a token and eight elements of each head
    int32_t run[kItems], token[kItems], first[kItems], second[kItems], pair[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const uint32_t at = tid + i * kRopeThreads, t = r.per_head.div(at);
        const int32_t u = (int32_t)(at - t * per_head);
        token[i] = (int32_t)min(t, 63u);
        run[i] = t < tokens ? runs.of[t] : -1;
        const bool turns = !values && u * 4 < r.n_pairs, halves = turns && !r.adjacent;
        pair[i] = turns ? u * 4 : -1;
        first[i] = halves ? u * 4 : u * 8;
        second[i] = halves ? u * 4 + r.n_pairs : u * 8 + 4;
    }
    const uint8_t* src = values ? r.v : r.k;
    const int64_t stride = values ? r.v_stride : r.k_stride;
    uint8_t* cache = values ? r.cache.v : r.cache.k;
    for (int32_t h = 0; h < heads; ++h) {
        float4 lo[kItems], hi[kItems];
        const uint8_t* from = src + (int64_t)(head0 + h) * head_dim * kSize;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            if (run[i] < 0) continue;
            const uint8_t* p = from + (token0 + token[i]) * stride;
            lo[i] = load4<kIn, kStream>(p + first[i] * kSize);
            hi[i] = load4<kIn, kStream>(p + second[i] * kSize);
        }
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            uint32_t most = 0;
            if (run[i] >= 0) {
                if (pair[i] >= 0) {
                    const uint32_t at = (uint32_t)token[i] * (uint32_t)r.n_pairs + (uint32_t)pair[i];
                    turn(lo[i], hi[i], *reinterpret_cast<const float4*>(sines + at), *reinterpret_cast<const float4*>(cosines + at),
                         r.adjacent);
                }
                most = max(magnitude(lo[i]), magnitude(hi[i]));
            }
            if (per_head % 4 == 0) {
                most = quad_max(most);
                if (run[i] >= 0 && (tid & 3) == 0) atomicMax(&runs.most[h][run[i]], most);
            } else if (run[i] >= 0) {
                atomicMax(&runs.most[h][run[i]], most);
            }
        }
        __syncthreads();
        uint8_t* to = cache + (int64_t)(head0 + h) * r.cache.head_stride;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            if (run[i] < 0) continue;
            const int32_t held = runs.held[run[i]];
            const float old = runs.old[h][run[i]], scale = new_scale(runs.most[h][run[i]], held, old);
            const float by = scale == scale ? 1.0f / scale : 0.0f;
            uint8_t* p = to + runs.place[token[i]];
            *reinterpret_cast<uint32_t*>(p + first[i]) = codes(lo[i], by);
            *reinterpret_cast<uint32_t*>(p + second[i]) = codes(hi[i], by);
            const int32_t u = (int32_t)(tid + i * kRopeThreads - r.per_head.div(tid + i * kRopeThreads) * per_head);
            const int32_t nth = token[i] - run[i];
            if (u == 0 && nth == 0) scale_of[runs.scale_at[run[i]] + h * a.scales.head_stride] = scale;
            if (held && scale > old) {  // not where either is NaN
                const float again = old / scale;
                for (int32_t t = nth; t < held; t += runs.count[run[i]]) {
                    u32x2* c = reinterpret_cast<u32x2*>(to + runs.block_at[run[i]] + t * r.cache.token_stride + u * 8);
                    const u32x2 v = *c;
                    *c = u32x2{scaled_codes(v[0], again), scaled_codes(v[1], again)};
                }
            }
        }
    }
}

template <int kIn, bool kStream, int kTokens, int kItems>
__global__ __launch_bounds__(kRopeThreads) void append_i8_kernel(AppendI8Args a, int head_dim, uint32_t beside) {
    if (blockIdx.x < a.kv_wgs) {
        const uint32_t part = blockIdx.x >> 1, chunk = a.by_head_groups.div(part);
        kv_workgroup<kIn, kStream, kItems>(a, head_dim, chunk, part - chunk * a.by_head_groups.d, blockIdx.x & 1);
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
    const uint32_t items = (a.chunk + (1u << a.scales.shift) - 1) * a.r.per_head.d;
    if (items <= 2 * kRopeThreads) return launch_items<kIn, 2>(a, head_dim, beside, stream, wgs, lds, s);
    if (items <= 4 * kRopeThreads) return launch_items<kIn, 4>(a, head_dim, beside, stream, wgs, lds, s);
    return launch_items<kIn, 8>(a, head_dim, beside, stream, wgs, lds, s);
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
