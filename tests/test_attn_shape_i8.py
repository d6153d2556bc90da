"""How decode attention over 8-bit integers divides a call, asked on the host: where rows in one
piece (a workgroup's, or a wave's) and shares of tiles were timed on MI355X and differ by more than
10 %, the faster is taken."""
from test_launch_rules import run_program

SHAPES = r"""
#include <cstdio>
#include <initializer_list>
#include "attn_decode_shape.hpp"
using namespace attn;

int main() {
    // rows of half to all of four tiles on 8 key heads; time of rows in one piece over that of shares
    struct { int rows, dim; double ratio; } uncut[] = {
        {40, 128, .71}, {70, 128, .68}, {129, 128, .96}, {200, 128, .80}, {257, 128, .99}, {40, 64, .83}, {70, 64, .78}, {129, 64, 1.07},
        {200, 64, .87}, {257, 64, 1.09}, {40, 256, .72}, {70, 256, .68}, {129, 256, 1.00}, {200, 256, .83}, {257, 256, 1.00}};
    for (const auto& u : uncut)
        if ((decode_whole(4, u.rows * 8) || decode_uncut_i8(4, u.rows, 8, kRound / 8, u.dim)) != (u.ratio < 1) &&
            (u.ratio < 0.91 || u.ratio > 1.1)) {
            printf("%d rows, dim %d: %g\n", u.rows, u.dim, u.ratio);
            return 1;
        }
    // a tile is about 8 KB of keys: other sub-tiles than the other byte caches'
    for (int dim : {64, 96, 128, 192, 256})
        if (decode_subtiles_i8(dim) * 32 * dim > 8192 || decode_subtiles_i8(dim) > decode_subtiles(dim, true)) return 2;
    // never beside whole rows; not where lengths may differ by more
    for (int dim : {64, 128, 256})
        for (int64_t pairs = 1; pairs < 10000; ++pairs)
            for (int most = 1; most < 40; ++most)
                if (decode_uncut_i8(most, pairs, 1, kRound, dim) && (decode_whole(most, pairs) || most > 4)) return 3;
    puts("ok");
    return 0;
}
"""


def test_division_of_a_call(tmp_path):
    run_program(tmp_path, "attn_shape_i8", SHAPES)
