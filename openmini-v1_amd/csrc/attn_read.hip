// Tokens of requests read out of a paged cache into dense rows (openmini_kv_read).
//
// An item is eight elements of one token and head, eight or sixteen bytes in; neighbouring lanes
// take neighbouring items, a thread the same item of its tokens, whose loads are all issued before
// the first is used.  A wave finds the tokens' places, a lane each, and leaves them in LDS.
//
// Bound by memory for long calls and by its three dependent loads (starts, page, elements) for short
// ones.  Measured (MI355X): 64 requests of 500 to 4000 tokens, 8 heads of 128, to fp16 113 us (656 MB, 5.8 TB/s),
// 16-bit and e4m3 caches to 16 bits at 5.8 and 5.7 TB/s, to fp32 348 us (1005 MB, 2.9 TB/s; of 16-bit caches 3.6); 300
// tokens to bf16 4.7 (in a trace 3.5); the last blocks of 200 requests in a trace 5.4, where a search of its own for each
// lane's run took 6.2.  One token a thread with its place worked out by itself took 177 and 8.2.
#include "attn_rope.hpp"
#include "attn_runs.hpp"

namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMostTokens = 64;  // of a workgroup

// Eight elements as they lie in the cache, and in 32 bits.
template <int kCache>
constexpr int kWords = kCache == OPENMINI_ATTN_F8_E4M3 || kCache == OPENMINI_ATTN_I8 ? 2 : 4;

template <int kCache>
__device__ __forceinline__ void unpack(const uint32_t* u, float scale, float4* lo, float4* hi) {
    if constexpr (kCache == OPENMINI_ATTN_F8_E4M3) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[0], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[0], true);
        const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[1], false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[1], true);
        *lo = make_float4(a[0], a[1], b[0], b[1]);
        *hi = make_float4(c[0], c[1], d[0], d[1]);
    } else if constexpr (kCache == OPENMINI_ATTN_I8) {
        *lo = make_float4((float)(int8_t)u[0], (float)(int8_t)(u[0] >> 8), (float)(int8_t)(u[0] >> 16), (float)(int8_t)(u[0] >> 24));
        *hi = make_float4((float)(int8_t)u[1], (float)(int8_t)(u[1] >> 8), (float)(int8_t)(u[1] >> 16), (float)(int8_t)(u[1] >> 24));
    } else if constexpr (kCache == OPENMINI_ATTN_BF16) {
        *lo = make_float4(__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xFFFF0000u), __uint_as_float(u[1] << 16),
                          __uint_as_float(u[1] & 0xFFFF0000u));
        *hi = make_float4(__uint_as_float(u[2] << 16), __uint_as_float(u[2] & 0xFFFF0000u), __uint_as_float(u[3] << 16),
                          __uint_as_float(u[3] & 0xFFFF0000u));
    } else {
        auto half = [&](int i) { return qmm::f16_bits_to_f32((uint16_t)(u[i / 2] >> (i & 1) * 16)); };
        *lo = make_float4(half(0), half(1), half(2), half(3));
        *hi = make_float4(half(4), half(5), half(6), half(7));
    }
    *lo = scaled(*lo, scale);
    *hi = scaled(*hi, scale);
    // products of 32 bits, whatever the output's type: not one instruction with the conversion
    asm("" : "+v"(lo->x), "+v"(lo->y), "+v"(lo->z), "+v"(lo->w), "+v"(hi->x), "+v"(hi->y), "+v"(hi->z), "+v"(hi->w));
}

template <int kOut, bool kStream>
__device__ __forceinline__ void store8(uint8_t* p, float4 lo, float4 hi) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    if constexpr (kOut == OPENMINI_ATTN_F32) {
        store<kStream>(p, f32x4{lo.x, lo.y, lo.z, lo.w});
        store<kStream>(p + 16, f32x4{hi.x, hi.y, hi.z, hi.w});
    } else if constexpr (kOut == OPENMINI_ATTN_BF16) {
        store<kStream>(p, u32x4{bf16_pair(lo.x, lo.y), bf16_pair(lo.z, lo.w), bf16_pair(hi.x, hi.y), bf16_pair(hi.z, hi.w)});
    } else {
        store<kStream>(p, u32x4{f16_pair(lo.x, lo.y), f16_pair(lo.z, lo.w), f16_pair(hi.x, hi.y), f16_pair(hi.z, hi.w)});
    }
}

// A workgroup takes kThreads items of kTokens tokens, or where a token has fewer all of
// kTokens * beside tokens; a thread one item, of kTokens tokens.
template <int kCache, int kOut, int kTokens, bool kStream>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a, uint32_t beside) {
    constexpr int kSize = kCache == OPENMINI_ATTN_F8_E4M3 || kCache == OPENMINI_ATTN_I8 ? 1 : 2, kOutSize = kOut == OPENMINI_ATTN_F32 ? 4 : 2;
    __shared__ int64_t place[kMostTokens], scale_at[kMostTokens];  // byte offset of a token's slot: -1 outside, -2 of no request
    const uint32_t tid = threadIdx.x, tokens = kTokens * beside;
    const int64_t token0 = (int64_t)blockIdx.x * tokens;
    if (tid < 64) {
        auto start = [&](uint32_t r) { return (uint32_t)max(a.starts[r], 0); };
        const int64_t token = token0 + tid;
        uint32_t run = find_run(a.requests, (uint32_t)token0, start);
        if (run == a.requests) run = 0;  // the first run begins behind the first token
        const bool mine = tid < tokens && token < a.tokens;
        // where the run and the 63 behind it end, a lane each: the lane's token is in the first that ends past
        // it; and the first tokens of the run and of those behind it, loaded beside
        int32_t from = a.starts[run], first = a.first ? a.first[run] : 0;
        const int32_t ends = a.starts[min(run + 1 + tid, a.requests)];
        const int32_t firsts = a.first ? a.first[min(run + 1 + tid, a.requests - 1)] : 0;
        uint32_t past = 0;  // runs that end before it
#pragma unroll
        for (uint32_t half = 32; half; half /= 2)
            if (__shfl(ends, (int)(past + half - 1)) <= token) past += half;
        const int behind = (int)max(past, 1u) - 1;
        const int32_t other_from = __shfl(ends, behind), other_first = __shfl(firsts, behind);
        int32_t to = __shfl(ends, (int)past);
        if (past) {
            from = other_from;
            first = other_first;
        }
        run = min(run + past, a.requests - 1);
        if (mine && to <= token && past == 63) {  // more runs than that
            for (uint32_t end = a.requests; end - run > 1;) {
                const uint32_t mid = run + (end - run) / 2;
                if (a.starts[mid] <= token)
                    run = mid;
                else
                    end = mid;
            }
            from = a.starts[run];
            to = a.starts[run + 1];
            first = a.first ? a.first[run] : 0;
        }
        int64_t at = -2, scale = 0;
        if (mine && token >= from && token < to) {
            at = -1;
            const int64_t pos = token - from + first;
            if (pos >= 0 && pos < a.max_len) {
                const uint32_t column = a.cache.page.div((uint32_t)pos), in_page = (uint32_t)pos - column * a.cache.page.d;
                const int32_t page = a.tables[run * a.table_stride + column];
                if ((uint32_t)page < a.cache.n_pages) {
                    at = page * a.cache.page_stride + in_page * a.cache.token_stride;
                    scale = page * a.scales.page_stride + (int64_t)(in_page >> a.scales.shift) * a.scales.block_stride;
                }
            }
        }
        place[tid] = at;
        if constexpr (kCache == OPENMINI_ATTN_I8) scale_at[tid] = scale;
    }
    __syncthreads();
    const uint32_t items = a.per_token.d, sub = beside > 1 ? a.per_token.div(tid) : 0, item = blockIdx.y * kThreads + tid - sub * items;
    if (sub >= beside || item >= items) return;
    const uint32_t h = a.per_head.div(item), u = item - h * a.per_head.d;
    const bool values = blockIdx.z || !a.k_out;
    const uint8_t* cache = (values ? a.cache.v : a.cache.k) + h * a.cache.head_stride + u * 8 * kSize;
    const float* scales = (values ? a.scales.v : a.scales.k) + h * a.scales.head_stride;
    const float whole = values ? a.cache.v_scale : a.cache.k_scale;
    const int64_t stride = values ? a.v_stride : a.k_stride;
    uint8_t* to = (values ? a.v_out : a.k_out) + (token0 + sub) * stride + (int64_t)item * 8 * kOutSize;
    typedef uint32_t words __attribute__((ext_vector_type(kWords<kCache>)));
    uint32_t raw[kTokens][kWords<kCache>];
    float scale[kTokens];
#pragma unroll
    for (int b = 0; b < kTokens; ++b) {
        const int64_t at = place[b * beside + sub];
        const words w = load<words, kStream>(cache + max(at, (int64_t)0));
#pragma unroll
        for (int i = 0; i < kWords<kCache>; ++i) raw[b][i] = w[i];
        scale[b] = whole;
        if constexpr (kCache == OPENMINI_ATTN_I8) scale[b] = scales[scale_at[b * beside + sub]];
    }
#pragma unroll
    for (int b = 0; b < kTokens; ++b, to += beside * stride) {
        const int64_t at = place[b * beside + sub];
        if (at == -2) continue;
        float4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (at >= 0) unpack<kCache>(raw[b], scale[b], &lo, &hi);
        store8<kOut, kStream>(to, lo, hi);
    }
}

template <int kCache, int kOut>
hipError_t launch_types(const ReadArgs& a, hipStream_t s) {
    // Eight tokens a thread, past the caches, where that leaves four workgroups to a CU; else two,
    // for the least latency.
    const uint32_t items = a.per_token.d, slices = (items + kThreads - 1) / kThreads, parts = a.k_out && a.v_out ? 2 : 1;
    uint32_t beside = items < kThreads ? kThreads / items : 1;
    const bool many = (a.tokens + 8 * beside - 1) / (8 * beside) * slices * parts >= 1024;
    const uint32_t tokens = many ? 8 : 2;
    if (beside > kMostTokens / tokens) beside = kMostTokens / tokens;
    const dim3 grid((unsigned)((a.tokens + tokens * beside - 1) / (tokens * beside)), slices, parts);
    if (many)
        hipLaunchKernelGGL((read_kernel<kCache, kOut, 8, true>), grid, dim3(kThreads), 0, s, a, beside);
    else
        hipLaunchKernelGGL((read_kernel<kCache, kOut, 2, false>), grid, dim3(kThreads), 0, s, a, beside);
    return hipGetLastError();
}

template <int kCache>
hipError_t launch_cache(const ReadArgs& a, hipStream_t s) {
    if (a.out_dtype == OPENMINI_ATTN_F32) return launch_types<kCache, OPENMINI_ATTN_F32>(a, s);
    if (a.out_dtype == OPENMINI_ATTN_BF16) return launch_types<kCache, OPENMINI_ATTN_BF16>(a, s);
    return launch_types<kCache, OPENMINI_ATTN_F16>(a, s);
}

}  // namespace

hipError_t launch_read(const ReadArgs& a, hipStream_t s) {
    switch (a.cache_dtype) {
    case OPENMINI_ATTN_F16: return launch_cache<OPENMINI_ATTN_F16>(a, s);
    case OPENMINI_ATTN_BF16: return launch_cache<OPENMINI_ATTN_BF16>(a, s);
    case OPENMINI_ATTN_F8_E4M3: return launch_cache<OPENMINI_ATTN_F8_E4M3>(a, s);
    case OPENMINI_ATTN_I8: return launch_cache<OPENMINI_ATTN_I8>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace attn
