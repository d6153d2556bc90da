// How decode attention divides a call: tiles, shares, and the rules for whole and uncut rows.
// Plain C++, asked by the host and by CPU tests.
#pragma once

#include <cstdint>

namespace attn {

constexpr int kDecodeWaves = 4;  // waves of a workgroup
// Keys that a wave takes at a time, in 32s: about 16 KB of keys and values.
constexpr int decode_subtiles(int head_dim, bool f8) {
    return f8 ? (head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 1) : head_dim <= 64 ? 2 : 1;
}
constexpr int kHeadTile = 16;    // query heads a workgroup serves (the MFMA's columns)
// Waves of a call, at most (one share each unless the units alone are more): one for each
// SIMD.  Two or three raise the bytes in flight past what the memory needs, and then equal
// shares end at different times (131071 keys, 8 heads of 128, bf16: 2048 waves 103 us, 1536
// 116, 1024 93).
constexpr int kRound = 1024;

// Whether workgroups take whole rows: `most` tiles in a row at most, by the table's columns
// and the window, and `pairs` of a row and a unit.  Up to two workgroups for each CU, and rows
// of up to 16 tiles, or 32 where the shares are no more than 16 for each pair either: two or
// four tiles for each of eight waves, and in 16-bit heads of 256, which have four waves, the limits
// are the same (8 pairs of 12 / 16 / 24 tiles .83 / .99 / 1.32 of the time of shares, 128 of 24 / 32
// .77 / .77).  Measured, whole rows against shares (us): 8 pairs of 300 keys, heads of 128, bf16
// 7.0 / 9.4, of 700 9.8 / 10.7, of 1000 12.5 / 10.9; 64 pairs of 1000 13.5 / 16.2, of 2000
// 22.6 / 18.5; 256 of up to 4000, heads of 64, 46.8 / 36.4; 512 of 400 15.1 / 20.4; 1024 of
// 200, e4m3, 16.6 / 16.3, of 60 14.3 / 9.5.
inline bool decode_whole(int64_t most, int64_t pairs) {
    return most == 1 ? pairs <= 256 : pairs <= 512 && most <= (pairs < 64 ? 16 : 32);
}

// Whether the shares are rows, as many to a wave as to any other whatever their lengths, so
// that no row is cut and there is no join: more pairs than workgroups take whole, of so few
// tiles that lengths do not differ by much, and `rows` not so little past a multiple of the
// `shares` that waves wait for the few with a row more.  That costs up to ceil(rows / shares) *
// most - ceil(rows * most / shares) tiles' time at the end, and the cut about 5 us for its join.
// Measured, uncut against shares of tiles (us): 1024 pairs of half to all of 4 tiles, heads of
// 128, bf16 11.3 / 16.9, of a twentieth to all 9.6 / 13.0; 2048 the same 20.8 / 27.7 and 15.1 /
// 17.1; of 8 tiles 39.2 / 43.1 and 23.5 / 23.7; 6000 of a twentieth to all of 4 tiles 40.3 / 39.9.
// 264 of one tile against whole rows 5.3 / 5.8, 128 5.2 / 5.3.  Past a multiple (time of uncut
// over cut, 8 key heads, half to all of 4 tiles, 1032 / 1104 / 1256 / 2056 / 2200 / 3104 pairs):
// heads of 128, bf16 1.03 1.02 .93 1.05 .97 .94, fp16 with a query head each 1.11 1.13 .98 1.07
// 1.01 1.04; of 64, bf16 1.12 1.15 1.04 1.09 1.04 1.08, e4m3 1.21 1.21 1.07 1.20 1.10 1.14; of 256,
// bf16 1.22 1.23 1.09 1.10 1.05 1.01 (of 3 tiles 1.14 1.15 .97 1.00 .99 1.03, but in heads of 128
// .97 .96 .83 .91 .92 .95).  One key head, whose join has a row for each share: heads of 128 .93
// .94 .85 .92 .85 .82, of 256 1.14 1.13 1.01 1.01 .94 .95, of 64 in e4m3 1.06 1.07 .95 1.06 .98 .98.
// So the rows are cut where 48 KB of tiles or more would be waited for, or 96 KB where there are one or
// two units; a tile of 128 keys, which the issue of instructions bounds, counts twice.
inline bool decode_uncut(int64_t most, int64_t rows, int64_t units, int64_t shares, int head_dim, bool f8) {
    const int64_t pairs = rows * units;
    if (most == 1) return pairs > 256;
    if (pairs <= 512 || most > (pairs <= 4096 ? 4 : 2)) return false;
    const int64_t tiles = (rows + shares - 1) / shares * most - (rows * most + shares - 1) / shares;
    const int sub = decode_subtiles(head_dim, f8), tile = 2 * 32 * sub * head_dim * (f8 ? 1 : 2) * (sub == 4 ? 2 : 1);
    return tiles * tile < (units > 2 ? 48 << 10 : 96 << 10);
}

}  // namespace attn
