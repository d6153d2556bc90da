"""Arrays of one call that share memory, in calls of include/openmini_kv_i8.h: refused before any
device work, and only where an element is shared."""
import ctypes

import pytest

from openmini_qmm import DType, _native
from test_attn_abi import BAD, _refused
from test_launch_rules import run_program

M = 1 << 20  # arrays lie this far apart


def _cache(**kw):
    a = dict(d_k=M, d_v=2 * M, dtype=DType.I8, kv_heads=2, head_dim=128, page_size=16, n_pages=4, page_stride=4096,
             token_stride=256, head_stride=128, k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return _native.KvCache(**a)


def _scales(**kw):
    a = dict(d_k=3 * M, d_v=4 * M, block=8, page_stride=4, block_stride=2, head_stride=1)
    a.update(kw)
    return _native.KvScales(**a)


# A rope of no pairs; refusals come before it is looked at, and calls of no tokens end behind that.
ROPE = ctypes.create_string_buffer(256)


def _append(cache, scales):
    args = _native.RopeAppendArgs(16 * M, 17 * M, 18 * M, 512, 256, 256, 19 * M, 512, DType.F32, DType.BF16, 0, 4, 20 * M, 0, 21 * M)
    return _native.lib().openmini_rope_append_i8(ctypes.cast(ROPE, ctypes.c_void_p), cache, scales, args, None)


def _taken(rc):
    """Past the checks: done (no tokens), or stopped for want of a GPU."""
    assert rc in (0, _native.ERR_HIP), (rc, _native.last_error())


@pytest.mark.parametrize("cache,scales,word", [
    ({}, dict(d_v=3 * M), "scales' d_k and d_v"), ({}, dict(d_v=3 * M + 4), "scales' d_k and d_v"), ({}, dict(d_k=4 * M + 60), "scales' d_k and d_v"),
    ({}, dict(d_k=4 * M - 4, page_stride=12, block_stride=6, head_stride=1), "scales' d_k and d_v"),
    (dict(d_v=M), {}, "cache's d_k and d_v"), (dict(d_v=M + 16), {}, "cache's d_k and d_v"), (dict(d_k=2 * M + 4 * 4096 - 16), {}, "cache's d_k and d_v"),
    (dict(d_v=M + 128, page_stride=8192, token_stride=512, head_stride=256, head_dim=256), {}, "cache's d_k and d_v"),
    (dict(page_stride=2048), {}, "two slots"), (dict(token_stride=0), {}, "two slots"), (dict(head_stride=64), {}, "two slots")])
def test_writes_that_meet(cache, scales, word):
    _refused(_append(_cache(**cache), _scales(**scales)), BAD, word)


@pytest.mark.parametrize("cache,scales", [
    ({}, {}), ({}, dict(d_v=3 * M + 64)), ({}, dict(d_k=4 * M + 64)),
    # keys and values, and their scales, element beside element, head beside head, token beside token, page beside page
    ({}, dict(d_v=3 * M + 4, page_stride=8, block_stride=4, head_stride=2)), ({}, dict(d_v=3 * M + 8, page_stride=8, block_stride=4, head_stride=1)),
    ({}, dict(d_v=3 * M + 16, page_stride=8, block_stride=2, head_stride=1)), ({}, dict(d_v=3 * M + 16, page_stride=8, block_stride=1, head_stride=2)),
    (dict(d_v=M + 128, page_stride=8192, token_stride=512, head_stride=256), {}), (dict(d_v=M + 256, page_stride=8192, token_stride=512), {}),
    (dict(d_v=M + 4096, page_stride=8192), {}), (dict(d_v=M + 2 * 2048, page_stride=8192, token_stride=128, head_stride=2048), {}),
    # codes and scales of a page side by side
    (dict(d_v=M + 4096, page_stride=8192 + 32), dict(d_k=M + 8192, d_v=M + 8208, page_stride=(8192 + 32) // 4)),
    # strides of axes of one do not matter
    (dict(n_pages=1, page_stride=0), dict(page_stride=0)), (dict(kv_heads=1, head_stride=0), dict(head_stride=0))])
def test_writes_beside_each_other(cache, scales):
    _taken(_append(_cache(**cache), _scales(**scales)))


def _read(**kw):
    a = dict(d_tables=5 * M, table_stride=4, max_pages=4, requests=2, d_starts=6 * M, d_first=7 * M, tokens=5, d_k_out=8 * M, d_v_out=9 * M,
             k_stride=256, v_stride=256, out_dtype=DType.BF16)
    a.update(kw)
    return _native.KvReadArgs(**a)


ROWS = 5 * 512  # bytes of an output's rows


@pytest.mark.parametrize("kw,word", [
    (dict(d_k_out=M + 16), "the cache"), (dict(d_v_out=M + 4 * 4096 - 16), "the cache"), (dict(d_k_out=2 * M - ROWS + 16), "the cache"),
    (dict(d_k_out=None, d_v_out=2 * M + 4096), "the cache"), (dict(d_v_out=3 * M), "the scales"), (dict(d_k_out=4 * M + 48), "the scales"),
    (dict(d_k_out=5 * M), "d_tables"), (dict(d_k_out=5 * M - ROWS + 16), "d_tables"), (dict(d_v_out=5 * M + 16), "d_tables"), (dict(d_v_out=6 * M), "d_starts"),
    (dict(d_k_out=7 * M), "d_first"), (dict(d_v_out=8 * M + 16), "d_k_out and d_v_out"), (dict(d_v_out=8 * M - ROWS + 16), "d_k_out and d_v_out"),
    (dict(d_v_out=8 * M + 512 - 16, k_stride=512, v_stride=512), "d_k_out and d_v_out"),
    (dict(d_v_out=8 * M + 512, k_stride=512, v_stride=768), "d_k_out and d_v_out"),
    (dict(d_k_out=M - (1 << 19), k_stride=1 << 19), "share memory"), (dict(d_k_out=16, k_stride=1 << 40, tokens=1 << 26), "share memory")])
def test_reads_over_what_they_read(kw, word):
    _refused(_native.lib().openmini_kv_read(_cache(), _scales(), _read(**kw), None), BAD, word)


@pytest.mark.parametrize("cache,kw", [
    ({}, {}), ({}, dict(d_k_out=M - ROWS)), ({}, dict(d_k_out=M + 4 * 4096)), ({}, dict(d_v_out=3 * M + 64)), ({}, dict(d_v_out=5 * M + 32)),
    ({}, dict(d_k_out=None, k_stride=0)), ({}, dict(d_v_out=None, v_stride=0)), ({}, dict(d_v_out=8 * M + ROWS)), ({}, dict(d_v_out=8 * M + 512, k_stride=512, v_stride=512)), ({}, dict(d_first=None, d_k_out=7 * M)),
    # a layer's pages between those of others: an output in another layer's part
    (dict(page_stride=1 << 17), dict(d_k_out=M + 4096)), (dict(page_stride=1 << 17), dict(d_k_out=M + (1 << 17) - ROWS))])
def test_reads_beside_what_they_read(cache, kw):
    """What stops the call is that this machine has no GPU."""
    if _native.lib().openmini_qmm_is_available():
        pytest.skip("the pointers are not memory")
    rc = _native.lib().openmini_kv_read(_cache(**cache), _scales(), _read(**kw), None)
    assert rc == _native.ERR_HIP, (rc, _native.last_error())


BOXES = r"""
#include <cstdio>
#include <random>
#include <set>
#include "attn_overlap.hpp"

// Every answer against the places themselves.
int main() {
    std::mt19937 rng(1);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    int nested = 0, met = 0;
    for (int n = 0; n < 20000; ++n) {
        attn::Axis axes[4] = {{1, pick(1, 4)}};
        int64_t reach = axes[0].count;
        for (int i = 1; i < 4; ++i) {
            axes[i] = {n % 5 ? reach + pick(0, 3) : pick(0, 12), pick(1, 4)};
            reach += axes[i].stride * (axes[i].count - 1);
        }
        for (int i = 3; i > 0; --i) std::swap(axes[i], axes[pick(0, i)]);
        const attn::Box<4> box(axes);
        std::multiset<int64_t> places;
        for (int a = 0; a < axes[0].count; ++a)
            for (int b = 0; b < axes[1].count; ++b)
                for (int c = 0; c < axes[2].count; ++c)
                    for (int d = 0; d < axes[3].count; ++d)
                        places.insert(a * axes[0].stride + b * axes[1].stride + c * axes[2].stride + d * axes[3].stride);
        bool twice = false;
        for (int64_t p : places) twice = twice || places.count(p) > 1;
        if (twice && box.nested) return 1;
        const int64_t last = *places.rbegin();
        nested += box.nested;
        for (int k = 0; k < 20; ++k) {
            const int64_t apart = (int64_t)(rng() % (unsigned)(2 * last + 9)) - last - 4;
            bool same = false;
            for (int64_t p : places) same = same || places.count(p + apart);
            if (box.nested && box.meets_itself(apart) != same) return 2;
            met += same;
            const int64_t from = (int64_t)(rng() % (unsigned)(last + 20)) - 10, to = from + pick(0, 3) * pick(0, 9);
            bool in = false;
            for (int64_t p : places) in = in || (p >= from && p < to);
            if (box.nested ? box.meets(from, to) != in : in && !box.meets(from, to)) return 3;
        }
    }
    if (nested < 10000 || met < 10000) return 4;
    puts("ok");
    return 0;
}
"""


def test_boxes(tmp_path):
    run_program(tmp_path, "boxes", BOXES)
