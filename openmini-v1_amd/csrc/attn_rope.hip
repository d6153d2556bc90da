// Rotary positions (openmini_rope_apply) and, fused with the cache write, those of a
// step's q and k (openmini_rope_append).
//
// Pair i of a token turns by the angle p f_i, p its position on the pair's axis.  In fp32
// that product loses the angle itself at long positions (2^-24 of 100000 revolutions is
// 0.04 radians), so the frequency is kept as a 64-bit fraction of a revolution: the
// integer product wraps at whole turns, which is the reduction, and its top bits give the
// quadrant and a remainder of at most an eighth of a turn, where sine and cosine are short
// series.  A workgroup makes the sines of its tokens once, in LDS, for all their heads.
//
// An item is eight elements of a head (four pairs, or eight that pass through), two loads
// and two stores of four; neighbouring lanes take neighbouring items.  Bound by memory for
// prompts and by latency for single tokens, whose heads are spread over workgroups (each
// making the token's sines again); the first items' loads are issued before the sines.
// Measured (MI355X): 16128 tokens of 16 heads of 128, fp32 to bf16 37 us, 5.3 TB/s read and
// written (a plain copy of as many bytes that converts alike 30 us); 8191 tokens of 32 + 64
// heads of 128 into an fp16 cache, all of it, 112 us, 5.4 TB/s; one token 2.8 - 3.4 us.
#include "attn_internal.hpp"

namespace attn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kBatch = 3;      // items a thread loads before it stores
constexpr int kMaxTokens = 8;  // tokens of a workgroup

// sin and cos of `phase` / 2^64 revolutions.  Series on [-pi/4, pi/4]: the first term left
// out is below 2e-9 (sine, x^11 / 11!) and 2e-10 (cosine, x^12 / 12!).
__device__ __forceinline__ void sin_cos(uint64_t phase, float* sine, float* cosine) {
    const uint32_t quadrant = (uint32_t)((phase + ((uint64_t)1 << 61)) >> 62);
    const int32_t rest = (int32_t)((phase - ((uint64_t)quadrant << 62)) >> 32);  // in [-2^29, 2^29]
    const float x = (float)rest * 1.46291807926715968e-9f;                       // 2 pi / 2^32
    const float z = x * x;
    const float s = x * (1.0f + z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880)))));
    const float c =
        1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const float a = quadrant & 1 ? c : s, b = quadrant & 1 ? s : c;
    *sine = quadrant & 2 ? -a : a;
    *cosine = (quadrant + 1) & 2 ? -b : b;
}

// kStream: loads and stores that leave the caches to others (what a prompt's call reads is
// not read again, and its q comes back from memory; the cache's lines stay).
template <class V, bool kStream>
__device__ __forceinline__ V load(const uint8_t* p) {
    if constexpr (kStream) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    return *reinterpret_cast<const V*>(p);
}
template <bool kStream, class V>
__device__ __forceinline__ void store(uint8_t* p, V v) {
    if constexpr (kStream)
        __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
    else
        *reinterpret_cast<V*>(p) = v;
}

template <int kType, bool kStream>
__device__ __forceinline__ float4 load4(const uint8_t* p) {
    if constexpr (kType == OPENMINI_ATTN_F32) {
        const f32x4 v = load<f32x4, kStream>(p);
        return make_float4(v[0], v[1], v[2], v[3]);
    } else {
        const u32x2 u = load<u32x2, kStream>(p);
        if constexpr (kType == OPENMINI_ATTN_BF16)
            return make_float4(__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xFFFF0000u), __uint_as_float(u[1] << 16),
                               __uint_as_float(u[1] & 0xFFFF0000u));
        else
            return make_float4(qmm::f16_bits_to_f32((uint16_t)u[0]), qmm::f16_bits_to_f32((uint16_t)(u[0] >> 16)),
                               qmm::f16_bits_to_f32((uint16_t)u[1]), qmm::f16_bits_to_f32((uint16_t)(u[1] >> 16)));
    }
}

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}
// Past the largest e4m3 value the conversion gives NaN: such values stop at it; NaN stays.
__device__ __forceinline__ float f8_range(float a) { return a != a ? a : fminf(fmaxf(a, -448.0f), 448.0f); }

// Four elements, each rounded once to the nearest even of the type.
template <bool kStream>
__device__ __forceinline__ void store4(uint8_t* p, int type, float4 v) {
    if (type == OPENMINI_ATTN_BF16) {
        store<kStream>(p, u32x2{bf16_pair(v.x, v.y), bf16_pair(v.z, v.w)});
    } else if (type == OPENMINI_ATTN_F16) {
        store<kStream>(p, u32x2{f16_pair(v.x, v.y), f16_pair(v.z, v.w)});
    } else if (type == OPENMINI_ATTN_F8_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(v.x), f8_range(v.y), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(v.z), f8_range(v.w), w, true);
        store<kStream>(p, w);
    } else {
        store<kStream>(p, f32x4{v.x, v.y, v.z, v.w});
    }
}

__device__ __forceinline__ int size_of(int type) {
    return type == OPENMINI_ATTN_F32 ? 4 : type == OPENMINI_ATTN_F8_E4M3 ? 1 : 2;
}

__device__ __forceinline__ float4 scaled(float4 v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }

// What an item is: its head (of q, k or v), and where its two fours of elements are.
struct Item {
    int32_t token, head, first, second, pair;  // token of the workgroup; pair < 0: passes through
    int32_t part;                              // 0 q, 1 k, 2 v
};

__device__ __forceinline__ Item item_of(const RopeArgs& a, uint32_t i) {
    Item t;
    t.token = (int32_t)a.per_token.div(i);
    const uint32_t in_token = i - (uint32_t)t.token * a.per_token.d;
    const uint32_t h = a.per_head.div(in_token);
    const int32_t u = (int32_t)(in_token - h * a.per_head.d);
    t.head = (int32_t)h;
    t.part = 0;
    if (t.head >= a.heads) {
        t.head -= a.heads;
        t.part = 1;
        if (t.head >= a.kv_heads) {
            t.head -= a.kv_heads;
            t.part = 2;
        }
    }
    const bool turns = t.part < 2 && u * 4 < a.n_pairs;
    t.pair = turns ? u * 4 : -1;
    const bool halves = turns && !a.adjacent;
    t.first = halves ? u * 4 : u * 8;
    t.second = halves ? u * 4 + a.n_pairs : u * 8 + 4;
    return t;
}

template <int kIn, bool kStream>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a, int head_dim, int wg_tokens, uint32_t step) {
    __shared__ __attribute__((aligned(16))) float sines[kMaxTokens * kMaxPairs], cosines[kMaxTokens * kMaxPairs];
    __shared__ int64_t places[kMaxTokens];  // byte offset of a token's slot, or -1
    constexpr int kSize = kIn == OPENMINI_ATTN_F32 ? 4 : 2;
    const uint32_t tid = threadIdx.x;
    const int64_t token0 = (int64_t)blockIdx.x * wg_tokens;
    const uint32_t mine = (uint32_t)min((int64_t)wg_tokens, a.tokens - token0);
    const uint32_t total = mine * a.per_token.d;
    const int y_size = size_of(a.y_dtype), c_size = size_of(a.cache_dtype);

    bool first_round = true;
    for (uint32_t i0 = blockIdx.y * kThreads; i0 < total; i0 += kBatch * step) {
        Item items[kBatch];
        float4 lo[kBatch], hi[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const uint32_t i = i0 + (uint32_t)b * step + tid;
            if (i >= total) continue;
            const Item t = items[b] = item_of(a, i);
            const int64_t token = token0 + t.token;
            const uint8_t* src = t.part == 0 ? a.x + token * a.x_stride : t.part == 1 ? a.k + token * a.k_stride
                                                                                       : a.v + token * a.v_stride;
            src += (int64_t)t.head * head_dim * kSize;
            lo[b] = load4<kIn, kStream>(src + t.first * kSize);
            hi[b] = load4<kIn, kStream>(src + t.second * kSize);
        }
        if (first_round) {
            first_round = false;
            for (uint32_t j = tid; j < mine * (uint32_t)a.n_pairs; j += kThreads) {
                const uint32_t t = a.by_pairs.div(j), i = j - t * a.by_pairs.d;
                const RopePair pair = a.pairs[i];
                const int32_t p = a.positions[pair.axis * a.position_stride + token0 + t];
                float s, c;
                sin_cos((uint64_t)(int64_t)p * pair.step, &s, &c);
                sines[t * kMaxPairs + i] = (a.inverse ? -s : s) * a.scale;
                cosines[t * kMaxPairs + i] = c * a.scale;
            }
            if (a.slots && tid < mine) {
                const int32_t s = a.slots[token0 + tid];
                int64_t place = -1;
                if (s >= 0 && (uint32_t)s < a.cache.slots) {
                    const uint32_t page = a.cache.page.div((uint32_t)s);
                    place = (int64_t)page * a.cache.page_stride +
                            (int64_t)((uint32_t)s - page * a.cache.page.d) * a.cache.token_stride;
                }
                places[tid] = place;
            }
            __syncthreads();
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i0 + (uint32_t)b * step + tid >= total) continue;
            const Item t = items[b];
            float4 x = lo[b], y = hi[b];
            if (t.pair >= 0) {
                const float4 s = *reinterpret_cast<const float4*>(&sines[t.token * kMaxPairs + t.pair]);
                const float4 c = *reinterpret_cast<const float4*>(&cosines[t.token * kMaxPairs + t.pair]);
                if (a.adjacent) {
                    const float4 p = x, q = y;
                    x = make_float4(p.x * c.x - p.y * s.x, p.x * s.x + p.y * c.x, p.z * c.y - p.w * s.y,
                                    p.z * s.y + p.w * c.y);
                    y = make_float4(q.x * c.z - q.y * s.z, q.x * s.z + q.y * c.z, q.z * c.w - q.w * s.w,
                                    q.z * s.w + q.w * c.w);
                } else {
                    const float4 p = x, q = y;
                    x = make_float4(p.x * c.x - q.x * s.x, p.y * c.y - q.y * s.y, p.z * c.z - q.z * s.z,
                                    p.w * c.w - q.w * s.w);
                    y = make_float4(p.x * s.x + q.x * c.x, p.y * s.y + q.y * c.y, p.z * s.z + q.z * c.z,
                                    p.w * s.w + q.w * c.w);
                }
            }
            if (t.part == 0) {
                uint8_t* dst = a.y + (token0 + t.token) * a.y_stride + (int64_t)t.head * head_dim * y_size;
                store4<kStream>(dst + t.first * y_size, a.y_dtype, x);
                store4<kStream>(dst + t.second * y_size, a.y_dtype, y);
            } else if (places[t.token] >= 0) {
                uint8_t* dst = (t.part == 1 ? a.cache.k : a.cache.v) + places[t.token] + t.head * a.cache.head_stride;
                const float over = t.part == 1 ? a.k_over : a.v_over;
                store4<false>(dst + t.first * c_size, a.cache_dtype, scaled(x, over));
                store4<false>(dst + t.second * c_size, a.cache_dtype, scaled(y, over));
            }
        }
    }
}

}  // namespace

template <int kIn>
static void launch_type(const RopeArgs& a, int head_dim, dim3 grid, int wg_tokens, bool stream, hipStream_t s) {
    if (stream)
        hipLaunchKernelGGL((rope_kernel<kIn, true>), grid, dim3(kThreads), 0, s, a, head_dim, wg_tokens, grid.y * kThreads);
    else
        hipLaunchKernelGGL((rope_kernel<kIn, false>), grid, dim3(kThreads), 0, s, a, head_dim, wg_tokens, grid.y * kThreads);
}

hipError_t launch_rope(const RopeArgs& a, int head_dim, hipStream_t s) {
    // Up to 2048 workgroups of one item a thread (single tokens: least latency), else
    // workgroups of about kBatch items a thread that stream.  MI355X, fp32 to bf16, plain
    // and four items against streaming and three: 16128 tokens of 16 heads 45.7 and 38.0 us
    // (5.2 TB/s), 4096 of 64 + 16 heads into an e4m3 cache 55.3 and 46.4, 8191 of 96 heads
    // into an fp16 cache 120 both (5.0 TB/s).
    const int64_t items = a.per_token.d;
    int64_t wg_tokens = 1, split = (items + kThreads - 1) / kThreads;
    const bool stream = a.tokens * split > 2048;
    if (stream) {
        wg_tokens = kBatch * kThreads / items;
        wg_tokens = wg_tokens < 1 ? 1 : wg_tokens > kMaxTokens ? kMaxTokens : wg_tokens;
        split = (items * wg_tokens + kBatch * kThreads - 1) / (kBatch * kThreads);
    }
    const dim3 grid((unsigned)((a.tokens + wg_tokens - 1) / wg_tokens), (unsigned)split);
    if (a.x_dtype == OPENMINI_ATTN_F32)
        launch_type<OPENMINI_ATTN_F32>(a, head_dim, grid, (int)wg_tokens, stream, s);
    else if (a.x_dtype == OPENMINI_ATTN_F16)
        launch_type<OPENMINI_ATTN_F16>(a, head_dim, grid, (int)wg_tokens, stream, s);
    else
        launch_type<OPENMINI_ATTN_BF16>(a, head_dim, grid, (int)wg_tokens, stream, s);
    return hipGetLastError();
}

}  // namespace attn
