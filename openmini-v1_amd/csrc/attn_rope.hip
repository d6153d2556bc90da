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
#include "attn_rope.hpp"

namespace attn {
namespace {

template <int kIn, bool kStream, int kTokens>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a, int head_dim, uint32_t beside) {
    rope_workgroup<kIn, kStream, kTokens>(a, head_dim, beside, blockIdx.x, blockIdx.y);
}

}  // namespace

template <int kIn>
static void launch_type(const RopeArgs& a, int head_dim, dim3 grid, uint32_t beside, bool stream, hipStream_t s) {
    const size_t lds = 2 * 4 * (size_t)beside * a.n_pairs;
    if (stream)
        hipLaunchKernelGGL((rope_kernel<kIn, true, batch_of(kIn)>), grid, dim3(kRopeThreads), batch_of(kIn) * lds, s, a, head_dim,
                           beside);
    else
        hipLaunchKernelGGL((rope_kernel<kIn, false, 1>), grid, dim3(kRopeThreads), lds, s, a, head_dim, beside);
}

hipError_t launch_rope(const RopeArgs& a, int head_dim, hipStream_t s) {
    // Up to 2048 workgroups of one token (or of those side by side) a thread, for the least
    // latency; else batch_of tokens a thread, past the caches.  MI355X, us, the latter with 1,
    // 2, 3 and 4 tokens: 16128 tokens of 16 heads, fp32 to bf16 38.4, 35.1, 35.8, 34.8, from
    // bf16 29.1, 26.6, 24.3, 23.2; 8191 of 96 heads into an fp16 cache 118.3, 113.8, 113.9,
    // 117.0 (the cache's lines past the caches too: 127); 128 threads 119, 512 112.
    const uint32_t items = a.per_token.d, slices = (items + kRopeThreads - 1) / kRopeThreads;
    uint32_t beside = 1;
    if (items < kRopeThreads) beside = kRopeThreads / items < kMostBeside ? kRopeThreads / items : kMostBeside;
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
