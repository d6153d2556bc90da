// Tokens of requests read out of a paged cache into dense rows (openmini_kv_read).
//
// An item is eight elements of one token and head; neighbouring lanes take neighbouring
// items.  Bound by memory.
#include "attn_rope.hpp"
#include "attn_runs.hpp"

namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kTokens = 16;  // of a workgroup

template <int kCache>
__device__ __forceinline__ void load8(const uint8_t* p, float scale, float4* lo, float4* hi) {
    if constexpr (kCache == OPENMINI_ATTN_F8_E4M3) {
        const u32x2 u = *reinterpret_cast<const u32x2*>(p);
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[0], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[0], true);
        const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[1], false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[1], true);
        *lo = make_float4(a[0], a[1], b[0], b[1]);
        *hi = make_float4(c[0], c[1], d[0], d[1]);
    } else if constexpr (kCache == OPENMINI_ATTN_I8) {
        const u32x2 u = *reinterpret_cast<const u32x2*>(p);
        *lo = make_float4((float)(int8_t)u[0], (float)(int8_t)(u[0] >> 8), (float)(int8_t)(u[0] >> 16), (float)(int8_t)(u[0] >> 24));
        *hi = make_float4((float)(int8_t)u[1], (float)(int8_t)(u[1] >> 8), (float)(int8_t)(u[1] >> 16), (float)(int8_t)(u[1] >> 24));
    } else {
        *lo = load4<kCache, false>(p);
        *hi = load4<kCache, false>(p + 8);
    }
    *lo = scaled(*lo, scale);
    *hi = scaled(*hi, scale);
}

template <int kCache>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
    constexpr int kSize = kCache == OPENMINI_ATTN_F8_E4M3 || kCache == OPENMINI_ATTN_I8 ? 1 : 2;
    __shared__ int64_t place[kTokens], scale_at[kTokens];  // byte offset of a token's slot: -1 outside, -2 of no request
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const int64_t token0 = (int64_t)blockIdx.x * kTokens;
    for (uint32_t t = tid >> 6; t < kTokens; t += kThreads / 64) {
        const int64_t token = token0 + t;
        if (token >= a.tokens) {
            if (lane == 0) place[t] = -2;
            continue;
        }
        const uint32_t run = find_run(a.requests, (uint32_t)token, [&](uint32_t r) { return (uint32_t)max(a.starts[r], 0); });
        if (lane) continue;
        int64_t at = -2;
        if (run < a.requests && token >= a.starts[run] && token < a.starts[run + 1]) {
            at = -1;
            const int64_t pos = token - a.starts[run] + (a.first ? a.first[run] : 0);
            if (pos >= 0 && pos < a.max_len) {
                const uint32_t column = a.cache.page.div((uint32_t)pos), in_page = (uint32_t)pos - column * a.cache.page.d;
                const int32_t page = a.tables[run * a.table_stride + column];
                if ((uint32_t)page < a.cache.n_pages) {
                    at = page * a.cache.page_stride + in_page * a.cache.token_stride;
                    if constexpr (kCache == OPENMINI_ATTN_I8)
                        scale_at[t] = page * a.scales.page_stride + (int64_t)(in_page >> a.scales.shift) * a.scales.block_stride;
                }
            }
        }
        place[t] = at;
    }
    __syncthreads();
    const int out_size = size_of(a.out_dtype);
    const bool values = blockIdx.y ? true : !a.k_out;
    uint8_t* out = values ? a.v_out : a.k_out;
    const int64_t stride = values ? a.v_stride : a.k_stride;
    const uint8_t* cache = values ? a.cache.v : a.cache.k;
    const float* scales = values ? a.scales.v : a.scales.k;
    const float whole = values ? a.cache.v_scale : a.cache.k_scale;
    for (uint32_t i = tid; i < kTokens * a.per_token.d; i += kThreads) {
        const uint32_t t = a.per_token.div(i), in_token = i - t * a.per_token.d, h = a.per_head.div(in_token), u = in_token - h * a.per_head.d;
        const int64_t at = place[t];
        if (at == -2) continue;
        float4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (at >= 0) {
            float scale = whole;
            if constexpr (kCache == OPENMINI_ATTN_I8) scale = scales[scale_at[t] + h * a.scales.head_stride];
            load8<kCache>(cache + at + h * a.cache.head_stride + u * 8 * kSize, scale, &lo, &hi);
        }
        uint8_t* to = out + (token0 + t) * stride + (int64_t)in_token * 8 * out_size;
        store4<false>(to, a.out_dtype, lo);
        store4<false>(to + 4 * out_size, a.out_dtype, hi);
    }
}

}  // namespace

hipError_t launch_read(const ReadArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.tokens + kTokens - 1) / kTokens), a.k_out && a.v_out ? 2 : 1);
    switch (a.cache_dtype) {
    case OPENMINI_ATTN_F16: hipLaunchKernelGGL(read_kernel<OPENMINI_ATTN_F16>, grid, dim3(kThreads), 0, s, a); break;
    case OPENMINI_ATTN_BF16: hipLaunchKernelGGL(read_kernel<OPENMINI_ATTN_BF16>, grid, dim3(kThreads), 0, s, a); break;
    case OPENMINI_ATTN_F8_E4M3: hipLaunchKernelGGL(read_kernel<OPENMINI_ATTN_F8_E4M3>, grid, dim3(kThreads), 0, s, a); break;
    case OPENMINI_ATTN_I8: hipLaunchKernelGGL(read_kernel<OPENMINI_ATTN_I8>, grid, dim3(kThreads), 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace attn
