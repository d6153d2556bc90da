// Decode attention on fp16 queries (fp16 or e4m3 caches), and the cut of long rows.
#include "attn_decode.hpp"

namespace attn {

hipError_t launch_decode_f16(const DecodeArgs& a, int head_dim, bool f8, hipStream_t s) {
    return launch_type<F16>(a, head_dim, f8, s);
}

namespace {
// Workgroups of a call that is cut: about two of eight waves (four of four) for each CU.
int64_t waves_of(int head_dim) { return head_dim <= 128 ? 8 : 4; }
int64_t target_of(int64_t units, int head_dim) {
    const int64_t round = 2 * 256 * 8 / waves_of(head_dim);
    static_assert(2 * 256 * 8 / 4 <= kRound, "the counters' region");
    return (round + units - 1) / units;
}
}  // namespace

DecodeShape decode_shape(int64_t rows, int kv_heads, int head_tiles, int head_dim, int64_t max_len) {
    DecodeShape s;
    s.target_parts = (uint32_t)target_of((int64_t)kv_heads * head_tiles, head_dim);
    s.min_tiles = (uint32_t)waves_of(head_dim);  // a tile for each wave
    // sums over rows of ceil(tiles / part_tiles) with part_tiles >= total / target_parts
    const int64_t tiles = (max_len + kTile - 1) / kTile + 1;
    const int64_t by_share = rows + s.target_parts, by_length = rows * ((tiles + s.min_tiles - 1) / s.min_tiles);
    s.max_parts = (uint32_t)(by_length < by_share ? by_length : by_share);
    return s;
}

// A row of n > 1 parts has more than (n - 1) part_tiles >= n / 2 part_tiles tiles.
int64_t decode_split_parts(int kv_heads, int head_tiles, int head_dim) {
    return 2 * target_of((int64_t)kv_heads * head_tiles, head_dim);
}

}  // namespace attn
