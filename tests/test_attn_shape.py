"""How decode attention divides a call (csrc/attn_decode_shape.hpp), asked on the host: where whole
rows, uncut rows and shares of tiles were timed on MI355X and differ by more than 10 %, the
faster is taken."""
from test_launch_rules import run_program

SHAPES = r"""
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include "attn_decode_shape.hpp"
using namespace attn;

int main() {
    // rows of half to all of `most` tiles; time of uncut rows over that of shares
    struct { int most, rows, units, dim, f8; double ratio; } uncut[] = {
        {4, 128, 8, 128, 0, 0.63}, {4, 256, 8, 128, 0, 0.77}, {4, 157, 8, 128, 0, 0.93}, {4, 388, 8, 128, 0, 0.94},
        {3, 129, 8, 128, 0, 0.97}, {3, 257, 8, 128, 0, 0.91}, {4, 33, 32, 128, 0, 1.18}, {4, 65, 32, 128, 0, 1.14},
        {4, 129, 8, 64, 0, 1.12}, {4, 257, 8, 64, 0, 1.09},
        {4, 129, 8, 64, 1, 1.21}, {4, 257, 8, 64, 1, 1.20}, {3, 129, 8, 64, 1, 1.11}, {2, 132, 8, 64, 1, 0.91}, {4, 128, 8, 64, 1, 0.77},
        {4, 132, 8, 128, 1, 1.07}, {2, 132, 8, 128, 1, 0.87},
        {4, 258, 4, 256, 0, 1.22}, {4, 514, 4, 256, 0, 1.10}, {3, 258, 4, 256, 0, 1.14}, {2, 264, 4, 256, 0, 0.88}, {4, 256, 4, 256, 0, 0.74},
        {4, 1025, 1, 128, 0, 0.93}, {4, 1250, 1, 128, 0, 0.85}, {4, 2049, 1, 128, 0, 0.92}, {4, 3100, 1, 128, 0, 0.82},
        {4, 1025, 1, 256, 0, 1.14}, {4, 1025, 1, 64, 1, 1.06}, {4, 513, 2, 256, 0, 1.19}, {4, 513, 2, 64, 1, 1.13},
    };
    for (const auto& u : uncut)
        if (decode_uncut(u.most, u.rows, u.units, kRound / u.units, u.dim, u.f8) != (u.ratio < 1) && (u.ratio < 0.91 || u.ratio > 1.1)) {
            printf("%d tiles, %d rows, %d units, dim %d, f8 %d: %g\n", u.most, u.rows, u.units, u.dim, u.f8, u.ratio);
            return 1;
        }
    // one tile: a wave a row, from 257 pairs on
    if (decode_uncut(1, 32, 8, 128, 128, false) || !decode_uncut(1, 33, 8, 128, 128, false) || !decode_uncut(1, 1000000, 8, 128, 128, false)) return 2;
    // never beside whole rows; not where lengths may differ by more
    for (int64_t pairs = 1; pairs < 10000; ++pairs)
        for (int most = 1; most < 40; ++most) {
            const bool u = decode_uncut(most, pairs, 1, kRound, 128, false);
            if (u && (decode_whole(most, pairs) || most > 4)) return 3;
        }
    // time of whole rows over that of shares, 16-bit heads of 256 (four waves a workgroup) and of 128
    struct { int most, pairs; double ratio; } whole[] = {{12, 8, 0.83}, {24, 8, 1.32}, {32, 32, 1.43}, {16, 64, 0.87}, {24, 128, 0.77},
                                                        {32, 128, 0.77}, {16, 512, 0.86}, {4, 512, 0.64}};
    for (const auto& w : whole)
        if (decode_whole(w.most, w.pairs) != (w.ratio < 1)) return 4;
    puts("ok");
    return 0;
}
"""


def test_division_of_a_call(tmp_path):
    run_program(tmp_path, "attn_shape", SHAPES)
