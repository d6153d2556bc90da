"""Scales of 8-bit caches at the ends of what they can be, and at ordinary sizes to a close bound."""
import numpy as np
import pytest

import attn_ref as ref
import kv_i8_ref as kv
import test_gpu_attn_decode_i8 as decode
import test_gpu_attn_prompt as prompt
from attn_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu
I8 = kv.I8

CODES = {"above": lambda rng, shape: rng.integers(1, 128, shape), "below": lambda rng, shape: -rng.integers(1, 128, shape),
         "both": lambda rng, shape: rng.integers(-127, 128, shape), "zero": lambda rng, shape: np.zeros(shape)}


def _positive(c, qmm):
    """Queries above zero, so that a key's score has the sign of its codes."""
    c.qb = ref.encode(np.abs(c.q) + 0.5, c.q_t)
    c.q = ref.decode(c.qb, c.q_t)
    c.queries(qmm)


@pytest.mark.parametrize("codes", sorted(CODES))
@pytest.mark.parametrize("lens,dim", [([100, 40], 64), ([700, 300], 128), ([9000, 60], 128), ([60] * 600, 64)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_decode_over_an_infinite_scale_of_keys(qmm, codes, lens, dim, bad):
    """The heads that see the block are NaN whatever the signs of its scores (all of them below zero
    would else be keys of no weight); rows before the block and the other heads are as ever.  Whole
    rows, rows cut into parts, and a wave to a row."""
    for q_t, out_t in ((BF16, F32), (F16, F16)):
        c = decode.Case(qmm, lens, 4, 2, dim, q_t, reqs=[0, 0, 0] + list(range(1, len(lens))), row_lens=[lens[0], 33, 32] + lens[1:], seed=dim)
        p = c.c
        page = p.tables[0, 2]  # keys 32 to 47 of request 0
        p.scales[0][page, 0, 0] = bad
        p.bits[0][page, :, 0] = CODES[codes](p.rng, (16, dim))
        p.upload(qmm)
        _positive(c, qmm)
        for scale in (None, -0.3):
            got = c.run(qmm, out_t, scale=scale)
            out = ref.decode(got[0], out_t)
            assert np.isnan(out[:2, :2]).all() and np.isnan(got[1][:2, :2]).all(), (np.isnan(out[:2, :2]).sum(), got[1][:2, :2])
            assert np.isfinite(out[:2, 2:]).all() and np.isfinite(got[1][:2, 2:]).all()
            c.check(got, out_t, scale=scale, skip=(0, 1) + tuple(range(8, len(c.reqs))))


@pytest.mark.parametrize("codes", sorted(CODES))
@pytest.mark.parametrize("dim,q_t,held,new", [(64, BF16, [20, 3], [50, 9]), (128, F16, [0, 0], [90, 40]), (128, BF16, [5000, 0], [4, 5]),
                                              (256, BF16, [10, 0], [60, 7])])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_prompts_over_an_infinite_scale_of_keys(qmm, codes, dim, q_t, held, new, bad):
    """Tokens from the block on are NaN in its heads, and with a window until it has passed; those
    before it and the other heads are as ever.  Tiles of a whole run, and keys split between workgroups."""
    for out_t, window in ((q_t, 0), (F32, 0), (q_t, 24)):
        c = prompt.Case(qmm, held, new, 4, 2, dim, q_t, I8, window=window, seed=dim)
        p = c.c
        first = (held[0] + new[0] // 2) // 16 * 16  # the block's first key
        page = p.tables[0, first // 16]
        p.scales[0][page, 0, 0] = bad
        p.bits[0][page, :, 0] = CODES[codes](p.rng, (16, dim))
        p.upload(qmm)
        _positive(c, qmm)
        seeing = [j for j in range(new[0]) if c.lens[j] > first and (not window or c.lens[j] - window < first + 16)]
        assert seeing
        for scale in (None, -0.3):
            got = c.run(qmm, out_t, scale=scale)
            out = ref.decode(got[0], out_t)
            for j in seeing:
                assert np.isnan(out[j, :2]).all() and np.isnan(got[1][j, :2]).all(), (j, np.isnan(out[j, :2]).sum(), got[1][j, :2])
                assert np.isfinite(out[j, 2:]).all() and np.isfinite(got[1][j, 2:]).all(), j
            c.check(got, out_t, scale=scale, skip=set(seeing))


@pytest.mark.parametrize("q_t", [BF16, F16])
@pytest.mark.parametrize("power", [100, 120, 124, 126, 127])
def test_prompts_over_large_scales_of_values(qmm, q_t, power):
    """Values of -1 to 1 times 2^power, all of them finite in fp32: correct up to 2^126, NaN past that (the
    scale's reciprocal is no normal number), never a number that is not the result."""
    c = prompt.Case(qmm, [0, 50], [40, 20], 4, 2, 64, q_t, I8, seed=power)
    p = c.c
    p.bits[1][:] = p.rng.integers(-1, 2, p.bits[1].shape)
    p.scales[1][np.isfinite(p.scales[1])] = 2.0 ** power
    p.upload(qmm)
    got = c.run(qmm, F32)
    out, lse = ref.decode(got[0], F32), got[1].astype(np.float64)
    for r, (first, n) in enumerate(c.runs):
        keys, values = p.tokens(r, range(max(c.lens[first:first + n])))
        for j in range(first, first + n):
            o, l, size, dots = ref.attention(c.q[j], keys[:c.lens[j]], values[:c.lens[j]], 0.125)
            d, e = prompt.bounds(o, size, dots, 2.0 ** power, 64, q_t, I8, F32, c.lens[j])
            if power <= 126:
                assert np.all(np.abs(out[j] - o) <= d) and np.all(np.abs(lse[j] - l) <= e + 2.0 ** -22 * np.abs(l)), j
            else:
                assert np.isnan(out[j]).all() and np.isnan(lse[j]).all(), j


@pytest.mark.parametrize("low,high", [(-60, 40), (-40, 30), (-40, 60)])
def test_prompts_over_scales_of_values_far_apart(qmm, low, high):
    """Up to 2^100: the keys of the least scales keep their weight among the others'."""
    for q_t, out_t in ((BF16, F32), (F16, F16), (BF16, BF16)):
        c = prompt.Case(qmm, [0, 90], [64, 30], 4, 2, 64, q_t, I8, seed=high, q_size=0.05)
        p = c.c
        for r in range(2):  # fp16 outputs: no more than they hold
            p.scales[1][p.tables[r, 0], 0] = 2.0 ** low
            p.scales[1][p.tables[r, 1:3], 0] = 2.0 ** (high if out_t != F16 else 5)
        p.upload(qmm)
        c.check(c.run(qmm, out_t), out_t)
