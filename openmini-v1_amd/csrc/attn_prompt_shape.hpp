// How attention of runs of query tokens divides a call.  Plain C++, asked by the host and by
// CPU tests.
#pragma once

#include <cstdint>

namespace attn {

constexpr int kWaveRows = 32;  // a wave's columns: query tokens times heads
constexpr int prompt_waves(int head_dim) { return head_dim <= 128 ? 8 : 4; }
constexpr int prompt_keys(int head_dim) { return head_dim <= 128 ? 64 : 32; }  // of a step
constexpr int prompt_rows(int head_dim) { return kWaveRows * prompt_waves(head_dim); }

// Pairs of a tile and a split, at most, where tiles are split.
constexpr int kPromptParts = 512;

// Workgroups to a tile's keys, for `wgs` tiles of which none sees more than `keys`: as many as
// make two workgroups for each CU, each of 512 keys at least.
inline int64_t prompt_splits(int64_t wgs, int64_t keys) {
    int64_t s = kPromptParts / wgs;
    if (s > keys / 512) s = keys / 512;
    return s > 1 ? s : 1;
}

}  // namespace attn
