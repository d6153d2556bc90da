"""How attention of runs divides a call (csrc/attn_prompt_shape.hpp), asked on the host."""
from test_launch_rules import run_program

SHAPES = r"""
#include <cstdio>
#include <initializer_list>
#include "attn_prompt_shape.hpp"
using namespace attn;

int main() {
    // splits fit the workspace and leave 256 keys each; tiles hold every row of every request
    for (int dim : {64, 96, 128, 192, 256})
        for (int64_t rows : {1, 5, 100, 1000, 20000, 1048576})
            for (int64_t requests : {1, 3, 300, 1048576})
                for (int kv : {1, 8, 32})
                    for (int group : {1, 5, 8, 300, 1024})
                        for (int64_t keys : {1, 511, 512, 5000, 131071, 2147483392}) {
                            const PromptShape p = prompt_shape(dim, rows, requests, kv, group, keys);
                            if (p.waves != 4 && (p.waves != 8 || dim > 128)) return 1;
                            if (p.heads * p.tokens > kWaveRows * p.waves || p.heads < 1 || p.tokens < 1 || p.heads * p.head_tiles < group) return 2;
                            if (p.units != (int64_t)kv * p.head_tiles) return 3;
                            // one run of all rows, and a token to each run
                            if (p.tiles * p.tokens < rows || (rows >= requests && p.tiles < requests)) return 9;
                            if (p.splits < 1 || (p.splits > 1 && (p.wgs() * p.splits > kPromptParts || keys / p.splits < 256))) return 4;
                            if (kWaveRows * p.waves > prompt_rows(dim)) return 5;
                        }
    // few rows under many keys are split, many rows are not, and take workgroups of eight waves
    if (prompt_shape(128, 4, 1, 8, 8, 60000).splits < 16 || prompt_shape(128, 8191, 1, 8, 8, 8191).splits != 1) return 6;
    if (prompt_shape(128, 8191, 1, 8, 8, 8191).waves != 8 || prompt_shape(128, 211, 1, 8, 8, 211).waves != 4) return 7;
    if (prompt_shape(128, 211, 1, 8, 8, 211).splits != 1) return 8;
    puts("ok");
    return 0;
}
"""


def test_division_of_a_call(tmp_path):
    run_program(tmp_path, "prompt_shape", SHAPES)
