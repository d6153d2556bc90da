// Attention of runs of bf16 query tokens.
#include "attn_prompt.hpp"

namespace attn {
hipError_t launch_prompt_bf16(const PromptArgs& a, int head_dim, int cache_dtype, bool out_f32, hipStream_t s) {
    return launch_prompt_type<BF16>(a, head_dim, cache_dtype, out_f32, s);
}
}  // namespace attn
