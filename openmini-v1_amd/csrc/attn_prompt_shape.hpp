// How attention of runs of query tokens divides a call.  Plain C++, asked by the host and by
// CPU tests.
#pragma once

#include <cstdint>

namespace attn {

constexpr int kWaveRows = 32;  // a wave's columns: query tokens times heads
constexpr int prompt_keys(int head_dim) { return head_dim <= 128 ? 64 : 32; }  // of a step

// Rows of a call's tiles, query tokens times heads: `heads` of a key head's `group`, and tokens.
struct PromptShape {
    int waves;  // 32 rows each
    int heads, tokens, head_tiles;
    int64_t tiles, units;  // of tokens, and of heads: workgroups of the call
    int64_t splits;        // workgroups that share a tile's keys
    int64_t wgs() const { return tiles * units; }
};

// Pairs of a tile and a split, at most, where tiles are split, and rows of a tile at most.
constexpr int kPromptParts = 512;
// Workgroups of four waves, at most, that have a CU each.
constexpr int prompt_alone(int head_dim) { return head_dim == 256 ? 384 : 256; }
constexpr int prompt_rows(int head_dim) { return head_dim <= 128 ? 256 : 128; }

inline PromptShape prompt_tiles(int waves, int64_t rows, int64_t requests, int kv_heads, int group) {
    PromptShape p;
    p.waves = waves;
    const int most = kWaveRows * waves;
    p.head_tiles = (group + most - 1) / most;
    p.heads = (group + p.head_tiles - 1) / p.head_tiles;
    p.tokens = most / p.heads;
    p.tiles = (rows + requests * (p.tokens - 1)) / p.tokens;
    p.units = (int64_t)kv_heads * p.head_tiles;
    p.splits = 1;
    return p;
}

// Time of a call, in steps of a workgroup of eight waves, of which a CU holds one (2 us): rounds of
// workgroups (the longest begin first, so a round need not be full to the last) times their steps,
// and 1.5 to begin and end; and a second launch that joins splits, whose parts are written and read at
// 4 TB/s.  Of four waves a CU holds one in .95 of the time, or two in 1.45 of it (1.2 in heads of 192 and
// 256, whose steps are half the keys).
// Measured (MI355X, us, four waves and eight): 200 tokens of 64 heads of 128 13.6 / 14.9, 3200 keys 97 /
// 104; a round of pairs of 66 steps 184, of eight waves 121.  64 tokens behind 8000 keys in 1, 4, 8, 16
// splits 251, 78, 51, 59; 512 behind 30000 in 2 and 3 530 and 690.
// Heads of 256 on fp16 caches with fp32 outputs have a CU each however many they are; the cost of more than
// prompt_alone counts them as the others.  The host's search takes up to 11 us (one tile over 131072 keys).
// Of several requests a tile each is taken to be half full; a round that this estimate fills to
// within 6 % is full or over in about half of the calls.
inline double prompt_cost(const PromptShape& p, int head_dim, int64_t rows, int64_t requests, int64_t steps, int64_t splits) {
    const int64_t spare = requests == 1 ? 2 * (p.tokens - 1) : requests * (p.tokens - 1);  // twice the rows that tiles lack
    const int64_t wgs = (2 * rows + spare + (requests > 1 ? 2 * p.tokens - 1 : 0)) / (2 * p.tokens) * p.units * splits;
    double each = 1, cus = 256;
    if (p.waves == 4) {
        const bool alone = wgs <= prompt_alone(head_dim);
        each = alone ? .95 : head_dim <= 128 ? 1.45 : 1.2;
        if (!alone) cus = 512;
    }
    const double full = wgs / cus, edge = requests == 1 ? 0 : .06;
    const double rounds = full <= 1 - edge ? 1 : full > 1 + edge || edge == 0 ? full + .3 : 1 + (full - 1 + edge) * (.3 + edge) / (2 * edge);
    const double join = splits > 1 ? 2.5 + 2.0 * wgs * p.heads * p.tokens * head_dim * 4 / (4e6 * 2) : 0;
    return rounds * ((double)((steps + splits - 1) / splits) + 1.5) * each + join;
}

// For rows that see up to `keys`.
inline PromptShape prompt_shape(int head_dim, int64_t rows, int64_t requests, int kv_heads, int group, int64_t keys) {
    const int64_t steps = (keys + prompt_keys(head_dim) - 1) / prompt_keys(head_dim);
    PromptShape best = {};
    double least = 0;
    for (int waves = 4; waves <= prompt_rows(head_dim) / kWaveRows; waves += 4) {
        PromptShape p = prompt_tiles(waves, rows, requests, kv_heads, group);
        for (int64_t s = 1; s == 1 || (s * p.wgs() <= kPromptParts && keys / s >= 256); ++s) {
            const double cost = prompt_cost(p, head_dim, rows, requests, steps, s);
            if (!best.waves || cost < least) {
                p.splits = s;
                best = p;
                least = cost;
            }
        }
    }
    return best;
}

}  // namespace attn
