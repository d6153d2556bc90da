// Decode attention on fp16 queries (fp16 or e4m3 caches), and the cut of a call into shares.
#include "attn_decode.hpp"

namespace attn {

hipError_t launch_decode_f16(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s) {
    return launch_type<F16>(a, head_dim, f8, s);
}

uint32_t decode_shares(int kv_heads, int head_tiles) {
    const int units = kv_heads * head_tiles;
    return units < kRound ? (uint32_t)(kRound / units) : 1;
}

}  // namespace attn
