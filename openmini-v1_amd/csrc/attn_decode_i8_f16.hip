// Decode attention on fp16 queries and caches of 8-bit integers.
#include "attn_decode.hpp"

namespace attn {
hipError_t launch_decode_i8_f16(const DecodeI8Args& a, int head_dim, hipStream_t s) {
    return launch_elem<F16, kI8>(a, head_dim, s);
}
}  // namespace attn
