// The second launch of attention of runs where tiles were split: the parts of a row are joined.
//
// Part i is a maximum m_i, a sum l_i and accumulators a_i relative to the maximum; with
// m = max m_i the row is sum a_i 2^(m_i - m) / sum l_i 2^(m_i - m).  A thread takes four
// dimensions of a row, the parts in their order, eight at a time.
#include "attn_prompt.hpp"

namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kDeep = 8;  // loads in flight

__global__ __launch_bounds__(kThreads) void prompt_join_kernel(PromptArgs a, int fours, int tile_rows, int out_dtype) {
    const uint32_t slot = a.by_units.div(blockIdx.x), unit = blockIdx.x - slot * a.by_units.d;
    const PromptTile tile = prompt_tile(a.starts, a.rows, a.requests, a.by_tokens, slot, unit, a.by_head_tiles, a.by_heads, a.group);
    const int at = (int)blockIdx.y * kThreads + (int)threadIdx.x, at_row = at / fours, d = at % fours * 4;
    const uint32_t token = a.by_heads.div((uint32_t)at_row), in_head = (uint32_t)at_row - token * a.by_heads.d;
    if (at_row >= tile_rows || token >= tile.tokens || in_head >= tile.heads) return;
    const int64_t entry = (int64_t)blockIdx.x * a.splits * tile_rows + at_row;
    float m = -INFINITY, l = 0;
    f32x4 v = {0, 0, 0, 0};
    for (uint32_t i0 = 0; i0 < a.splits; i0 += kDeep) {
        float2 ml[kDeep];
        f32x4 part[kDeep];
#pragma unroll
        for (uint32_t k = 0; k < kDeep; ++k) {
            const int64_t at = entry + (int64_t)min(i0 + k, a.splits - 1) * tile_rows;
            ml[k] = a.part_ml[at];
            part[k] = *reinterpret_cast<const f32x4*>(a.part_acc + at * fours * 4 + d);
        }
#pragma unroll
        for (uint32_t k = 0; k < kDeep; ++k) {
            if (i0 + k >= a.splits) break;
            const float to = fmaxf(m, ml[k].x), f0 = exp2_of(m - above(to)), f1 = exp2_of(ml[k].x - above(to));
            v = v * f0 + part[k] * f1;
            l = l * f0 + ml[k].y * f1;
            m = to;
        }
    }
    v *= l > 0 || l != l ? a.cache.v_scale / l : 0.0f;
    const uint32_t row = tile.token0 + token, head = tile.head0 + in_head;
    uint8_t* out = a.out + row * a.out_stride;
    const int64_t to = (int64_t)head * fours * 4 + d;
    if (out_dtype == OPENMINI_ATTN_F32)
        *reinterpret_cast<f32x4*>(out + to * 4) = v;
    else if (out_dtype == OPENMINI_ATTN_BF16)
        *reinterpret_cast<uint2*>(out + to * 2) = make_uint2(BF16::pair(v[0], v[1]), BF16::pair(v[2], v[3]));
    else
        *reinterpret_cast<uint2*>(out + to * 2) = make_uint2(F16::pair(v[0], v[1]), F16::pair(v[2], v[3]));
    if (a.lse && d == 0) a.lse[(int64_t)row * a.q_heads + head] = log_sum(m, l);
}

}  // namespace

hipError_t launch_prompt_join(const PromptArgs& a, int head_dim, int out_dtype, hipStream_t s) {
    const int fours = head_dim / 4, rows = kWaveRows * a.waves;
    hipLaunchKernelGGL(prompt_join_kernel, dim3(a.tiles * a.by_units.d, (unsigned)((rows * fours + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                       s, a, fours, rows, out_dtype);
    return hipGetLastError();
}

}  // namespace attn
