"""How attention of runs divides a call (csrc/attn_prompt_shape.hpp), asked on the host."""
from test_launch_rules import run_program

SHAPES = r"""
#include <cstdio>
#include <initializer_list>
#include "attn_prompt_shape.hpp"
using namespace attn;

int main() {
    // parts never exceed the workspace, and none has fewer than 512 keys on average
    for (int64_t wgs = 1; wgs < 3000; ++wgs)
        for (int64_t keys : {1, 511, 512, 1023, 1024, 5000, 131071, 2147483392}) {
            const int64_t s = prompt_splits(wgs, keys);
            if (s < 1 || (s > 1 && (wgs * s > kPromptParts || keys / s < 512))) return 1;
        }
    if (prompt_splits(8, 131071) != 64 || prompt_splits(8, 1023) != 1 || prompt_splits(300, 1 << 20) != 1) return 2;
    for (int d : {64, 96, 128, 192, 256})
        if (prompt_rows(d) != 32 * prompt_waves(d) || prompt_keys(d) % 32) return 3;
    puts("ok");
    return 0;
}
"""


def test_division_of_a_call(tmp_path):
    run_program(tmp_path, "prompt_shape", SHAPES)
