// The second launch of decode attention: the parts of rows that were cut are joined.
//
// Part i of a row is a maximum m_i, a sum l_i and accumulators a_i relative to the maximum;
// with m = max m_i the row is sum a_i 2^(m_i - m) / sum l_i 2^(m_i - m).  A workgroup takes
// some heads of a row; its threads are groups that take every groups-th part, a thread four
// dimensions, kDeep loads in flight, and the groups are joined in order.
//
// Bound by latency: a launch and two loads one after the other, of lines that other XCDs
// wrote; 4 to 6 us (131071 keys of one row, 128 parts of 64 heads of 128: 5.6).  A launch of
// its own and not the end of the first: there, waves that joined by pairs as they ended,
// through device-scope stores and loads, took longer on every call (one row of 300 keys 13.2
// against 9.3 us, of 131071 105 against 99.7, 64 rows in a window 33.8 against 30.8).
#include "attn_internal.hpp"
#include "qmm_device.hpp"

namespace attn {
namespace {

using qmm::f32x4;
constexpr int kThreads = 256;

__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.0f : m; }

struct Joined {
    f32x4 v = {0, 0, 0, 0};
    float m = -INFINITY, l = 0;
    __device__ __forceinline__ void add(f32x4 pv, float pm, float pl) {
        const float to = fmaxf(m, pm), f0 = __builtin_amdgcn_exp2f(m - above(to)), f1 = __builtin_amdgcn_exp2f(pm - above(to));
        v = v * f0 + pv * f1;
        l = l * f0 + pl * f1;
        m = to;
    }
};

template <uint32_t kDeep>
__global__ __launch_bounds__(kThreads) void join_kernel(const Split* __restrict__ split, const float* __restrict__ part_acc,
                                                        const float2* __restrict__ part_ml, uint8_t* __restrict__ out,
                                                        float* __restrict__ lse, int64_t out_stride, int q_heads, int wg_heads,
                                                        int fours, float v_scale, int out_dtype) {
    __shared__ f32x4 sum_v[kThreads];
    __shared__ float sum_m[kThreads], sum_l[kThreads];
    const Split row = split[blockIdx.x];
    if (row.parts <= 1) return;
    const int head0 = blockIdx.y * wg_heads, outs = wg_heads * fours, groups = kThreads / outs;
    const int tid = threadIdx.x, grp = tid / outs, o = tid - grp * outs, head = head0 + o / fours, d = o % fours * 4;
    const bool active = grp < groups && head < q_heads;
    Joined j;
    if (active) {
        for (uint32_t i0 = grp; i0 < row.parts; i0 += kDeep * groups) {
            f32x4 pv[kDeep];
            float2 pml[kDeep];
#pragma unroll
            for (uint32_t k = 0; k < kDeep; ++k) {
                const uint32_t i = min(i0 + k * groups, row.parts - 1);
                const int64_t entry = (int64_t)(2 * (row.first_share + i) + (i == 0)) * q_heads + head;
                pml[k] = part_ml[entry];
                pv[k] = *reinterpret_cast<const f32x4*>(part_acc + (entry * fours) * 4 + d);
            }
#pragma unroll
            for (uint32_t k = 0; k < kDeep; ++k)
                if (i0 + k * groups < row.parts) j.add(pv[k], pml[k].x, pml[k].y);
        }
    }
    if (groups > 1) {
        sum_v[tid] = j.v;
        sum_m[tid] = j.m;
        sum_l[tid] = j.l;
        __syncthreads();
        if (active && grp == 0)
            for (int k = 1; k < groups; ++k) j.add(sum_v[k * outs + o], sum_m[k * outs + o], sum_l[k * outs + o]);
    }
    if (!active || grp) return;
    const f32x4 v = j.v * (j.l > 0 || j.l != j.l ? v_scale / j.l : 0.0f);
    uint8_t* to = out + row.row * out_stride;
    const int64_t at = (int64_t)head * fours * 4 + d;
    if (out_dtype == OPENMINI_ATTN_F32) {
        *reinterpret_cast<f32x4*>(to + at * 4) = v;
    } else if (out_dtype == OPENMINI_ATTN_BF16) {
        typedef __bf16 v4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4*>(to + at * 2) = v4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    } else {
        typedef _Float16 v4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4*>(to + at * 2) = v4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    }
    if (lse && d == 0)
        lse[(int64_t)row.row * q_heads + head] = log_sum(j.m, j.l);
}

}  // namespace

hipError_t launch_join(const DecodeArgs& a, int head_dim, int out_dtype, hipStream_t s) {
    const uint32_t rows = a.by_row ? a.n_rows : a.launch_shares;
    // Parts of a row on average: all shares over all rows, and a cut at both ends.  Groups of
    // threads enough to leave each two of them, by fewer heads in a workgroup, down to one;
    // then a thread takes sixteen at a time (it loads the last part again past the end, so
    // not where there are few).
    const int fours = head_dim / 4;
    const int64_t parts = a.launch_shares / a.n_rows + 1;
    int wg_heads = kThreads / fours < a.q_heads ? kThreads / fours : a.q_heads;
    while (wg_heads > 1 && 2 * (kThreads / (wg_heads * fours)) < parts) wg_heads = (wg_heads + 1) / 2;
    const bool few = 2 * (kThreads / (wg_heads * fours)) >= parts;
    const dim3 grid(rows, (a.q_heads + wg_heads - 1) / wg_heads);
    if (few)
        hipLaunchKernelGGL(join_kernel<2>, grid, dim3(kThreads), 0, s, a.split, a.part_acc, a.part_ml, a.out, a.lse,
                           a.out_stride, a.q_heads, wg_heads, fours, a.cache.v_scale, out_dtype);
    else
        hipLaunchKernelGGL(join_kernel<16>, grid, dim3(kThreads), 0, s, a.split, a.part_acc, a.part_ml, a.out, a.lse,
                           a.out_stride, a.q_heads, wg_heads, fours, a.cache.v_scale, out_dtype);
    return hipGetLastError();
}

}  // namespace attn
