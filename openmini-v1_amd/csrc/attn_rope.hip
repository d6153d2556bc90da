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
// and two stores of four; neighbouring lanes take neighbouring items.  A thread takes the
// same item of its tokens, so what an item is, is worked out once.  Bound by memory for
// prompts and by latency for single tokens, whose heads are spread over workgroups (each
// making the token's sines again); the loads are issued before the sines.
// Measured (MI355X): 16128 tokens of 16 heads of 128, fp32 to bf16 35 us, 5.6 TB/s read and
// written (a copy alone that converts alike, in the same pieces, 31); 8191 tokens of 32 + 64
// heads of 128 into an fp16 cache 114 us, 5.3 TB/s (the copy 93); one token 2.8 - 3.4 us.
#include "attn_internal.hpp"

namespace attn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
// Tokens of a thread where a call streams: 64 bytes of loads.
constexpr int batch_of(int in) { return in == OPENMINI_ATTN_F32 ? 2 : 4; }
constexpr uint32_t kMostBeside = 32;  // tokens side by side in a workgroup
static_assert(4 * kMostBeside <= kThreads, "a thread to each token's slot");

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
    int32_t head, first, second, pair;  // pair < 0: passes through
    int32_t part;                       // 0 q, 1 k, 2 v
};

__device__ __forceinline__ Item item_of(const RopeArgs& a, uint32_t i) {
    Item t;
    const uint32_t h = a.per_head.div(i);
    const int32_t u = (int32_t)(i - h * a.per_head.d);
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

// A workgroup takes kThreads items of kTokens tokens, or where a token has fewer all of
// kTokens * beside tokens; a thread one item, of kTokens tokens.
template <int kIn, bool kStream, int kTokens>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a, int head_dim, uint32_t beside) {
    extern __shared__ __attribute__((aligned(16))) float sines[];  // [tokens][pairs], and as many cosines
    __shared__ int64_t places[kTokens * kMostBeside];              // byte offset of a token's slot, or -1
    constexpr int kSize = kIn == OPENMINI_ATTN_F32 ? 4 : 2;
    const uint32_t tid = threadIdx.x, items = a.per_token.d;
    const int64_t token0 = (int64_t)blockIdx.x * (kTokens * beside);
    const uint32_t mine = (uint32_t)min((int64_t)(kTokens * beside), a.tokens - token0);
    const int y_size = size_of(a.y_dtype), c_size = size_of(a.cache_dtype);
    float* cosines = sines + kTokens * beside * a.n_pairs;

    const uint32_t sub = beside > 1 ? a.per_token.div(tid) : 0, item = blockIdx.y * kThreads + tid - sub * items;
    const bool active = sub < beside && item < items;
    Item t = {};
    float4 lo[kTokens], hi[kTokens];
    if (active) {
        t = item_of(a, item);
        const int64_t stride = t.part == 0 ? a.x_stride : t.part == 1 ? a.k_stride : a.v_stride;
        const uint8_t* src = (t.part == 0 ? a.x : t.part == 1 ? a.k : a.v) + (token0 + sub) * stride + (int64_t)t.head * head_dim * kSize;
#pragma unroll
        for (int b = 0; b < kTokens; ++b, src += beside * stride) {
            if (b * beside + sub >= mine) break;
            lo[b] = load4<kIn, kStream>(src + t.first * kSize);
            hi[b] = load4<kIn, kStream>(src + t.second * kSize);
        }
    }
    for (uint32_t j = tid; j < mine * (uint32_t)a.n_pairs; j += kThreads) {
        const uint32_t token = a.by_pairs.div(j), i = j - token * a.by_pairs.d;
        const RopePair pair = a.pairs[i];
        const int32_t p = a.positions[pair.axis * a.position_stride + token0 + token];
        float s, c;
        sin_cos((uint64_t)(int64_t)p * pair.step, &s, &c);
        sines[j] = (a.inverse ? -s : s) * a.scale;
        cosines[j] = c * a.scale;
    }
    if (a.slots && tid < mine) {
        const int32_t s = a.slots[token0 + tid];
        int64_t place = -1;
        if (s >= 0 && (uint32_t)s < a.cache.slots) {
            const uint32_t page = a.cache.page.div((uint32_t)s);
            place = (int64_t)page * a.cache.page_stride + (int64_t)((uint32_t)s - page * a.cache.page.d) * a.cache.token_stride;
        }
        places[tid] = place;
    }
    __syncthreads();
    if (!active) return;
    uint8_t* y_row = a.y + (token0 + sub) * a.y_stride + (int64_t)t.head * head_dim * y_size;
    uint8_t* c_row = (t.part == 1 ? a.cache.k : a.cache.v) + t.head * a.cache.head_stride;
    const float over = t.part == 1 ? a.k_over : a.v_over;
#pragma unroll
    for (int b = 0; b < kTokens; ++b, y_row += beside * a.y_stride) {
        const uint32_t token = b * beside + sub;
        if (token >= mine) break;
        float4 x = lo[b], y = hi[b];
        if (t.pair >= 0) {
            const uint32_t at = token * (uint32_t)a.n_pairs + (uint32_t)t.pair;
            const float4 s = *reinterpret_cast<const float4*>(sines + at), c = *reinterpret_cast<const float4*>(cosines + at);
            const float4 p = x, q = y;
            if (a.adjacent) {
                x = make_float4(p.x * c.x - p.y * s.x, p.x * s.x + p.y * c.x, p.z * c.y - p.w * s.y, p.z * s.y + p.w * c.y);
                y = make_float4(q.x * c.z - q.y * s.z, q.x * s.z + q.y * c.z, q.z * c.w - q.w * s.w, q.z * s.w + q.w * c.w);
            } else {
                x = make_float4(p.x * c.x - q.x * s.x, p.y * c.y - q.y * s.y, p.z * c.z - q.z * s.z, p.w * c.w - q.w * s.w);
                y = make_float4(p.x * s.x + q.x * c.x, p.y * s.y + q.y * c.y, p.z * s.z + q.z * c.z, p.w * s.w + q.w * c.w);
            }
        }
        if (t.part == 0) {
            store4<kStream>(y_row + t.first * y_size, a.y_dtype, x);
            store4<kStream>(y_row + t.second * y_size, a.y_dtype, y);
        } else if (places[token] >= 0) {
            uint8_t* dst = c_row + places[token];
            store4<false>(dst + t.first * c_size, a.cache_dtype, scaled(x, over));
            store4<false>(dst + t.second * c_size, a.cache_dtype, scaled(y, over));
        }
    }
}

}  // namespace

template <int kIn>
static void launch_type(const RopeArgs& a, int head_dim, dim3 grid, uint32_t beside, bool stream, hipStream_t s) {
    const size_t lds = 2 * 4 * (size_t)beside * a.n_pairs;
    if (stream)
        hipLaunchKernelGGL((rope_kernel<kIn, true, batch_of(kIn)>), grid, dim3(kThreads), batch_of(kIn) * lds, s, a, head_dim,
                           beside);
    else
        hipLaunchKernelGGL((rope_kernel<kIn, false, 1>), grid, dim3(kThreads), lds, s, a, head_dim, beside);
}

hipError_t launch_rope(const RopeArgs& a, int head_dim, hipStream_t s) {
    // Up to 2048 workgroups of one token (or of those side by side) a thread, for the least
    // latency; else batch_of tokens a thread, past the caches.  MI355X, us, the latter with 1,
    // 2, 3 and 4 tokens: 16128 tokens of 16 heads, fp32 to bf16 38.4, 35.1, 35.8, 34.8, from
    // bf16 29.1, 26.6, 24.3, 23.2; 8191 of 96 heads into an fp16 cache 118.3, 113.8, 113.9,
    // 117.0 (the cache's lines past the caches too: 127); 128 threads 119, 512 112.
    const uint32_t items = a.per_token.d, slices = (items + kThreads - 1) / kThreads;
    uint32_t beside = 1;
    if (items < kThreads) beside = kThreads / items < kMostBeside ? kThreads / items : kMostBeside;
    const bool stream = (a.tokens + beside - 1) / beside * slices > 2048;
    const int64_t tokens = stream ? (int64_t)batch_of(a.x_dtype) * beside : beside;
    const unsigned groups = (unsigned)((a.tokens + tokens - 1) / tokens);
    const dim3 grid(groups, slices);
    if (a.x_dtype == OPENMINI_ATTN_F32)
        launch_type<OPENMINI_ATTN_F32>(a, head_dim, grid, beside, stream, s);
    else if (a.x_dtype == OPENMINI_ATTN_F16)
        launch_type<OPENMINI_ATTN_F16>(a, head_dim, grid, beside, stream, s);
    else
        launch_type<OPENMINI_ATTN_BF16>(a, head_dim, grid, beside, stream, s);
    return hipGetLastError();
}

}  // namespace attn
