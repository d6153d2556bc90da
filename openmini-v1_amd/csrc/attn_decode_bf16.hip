// Decode attention on bf16 queries (bf16 or e4m3 caches).
#include "attn_decode.hpp"

namespace attn {
hipError_t launch_decode_bf16(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s) {
    return launch_type<BF16>(a, head_dim, f8, s);
}
}  // namespace attn
