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


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_scales_of_values_that_are_not_finite(qmm, bad):
    """The heads that see the block are NaN, in decode and in prompt attention alike; rows before it and
    the other heads are as ever."""
    for q_t, out_t in ((BF16, F32), (F16, F16)):
        d = decode.Case(qmm, [100], 4, 2, 64, q_t, reqs=[0, 0, 0], row_lens=[100, 33, 32], seed=3)
        c = prompt.Case(qmm, [20], [40], 4, 2, 64, q_t, I8, seed=4)
        for case in (d, c):
            p = case.c
            p.scales[1][p.tables[0, 2], 0, 0] = bad  # values 32 to 47
            p.upload(qmm)
            seeing = [j for j, n in enumerate((d.row_lens if case is d else c.lens[:40])) if n > 32]
            got = case.run(qmm, out_t)
            out = ref.decode(got[0], out_t)
            assert seeing and np.isnan(out[seeing, :2]).all() and np.isfinite(out[seeing, 2:]).all(), (case is d, np.isnan(out[seeing, :2]).sum())
            case.check(got, out_t, skip=set(seeing))


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


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_t", [BF16, F16])
def test_prompts_over_two_blocks(qmm, dim, q_t):
    """Rows that see two blocks of 16 keys, scores of 0, all keys of a block alike, value scales of 2^-8
    to 2^-3, outputs of 32 bits: what the scales' way through the exponent costs, and next to nothing
    else (sums of 16 equal products are exact, and three bf16 parts leave 2^-24).  In units of 2^-24: a
    base-2 logarithm of less than 8, off by at most one unit in its last place, 8, two of them; their
    difference, of less than 8, by half of one, 4: an exponent is off by 20, a probability by 20 log 2
    = 14 and the exponential's 2.  A sum of probabilities by as much and the reciprocals' 2; one of each
    for its addition, the division and the product, 3.  16 + 18 + 3 and 1 for the parts: 38 of sum p |v|.
    lse: 18, and 3 numbers of less than 16 added, 8 each."""
    rng, n, kv_heads = np.random.default_rng(dim + q_t), 60, 8
    c = prompt.Case(qmm, [30] * n, [2] * n, kv_heads, kv_heads, dim, q_t, I8, lens=[32] * (2 * n), seed=dim, q_size=0.0)
    p = c.c
    for r in range(n):
        for b in range(2):
            page = p.tables[r, b]
            p.scales[1][page, 0] = (2.0 ** rng.uniform(-8, -3, kv_heads)).astype(np.float32)
            p.bits[1][page] = rng.integers(-127, 128, (kv_heads, dim))
    p.upload(qmm)
    got = c.run(qmm, F32)
    out, lse = ref.decode(got[0], F32), got[1].astype(np.float64)
    worst = 0.0
    for r in range(n):
        a, b = (p.bits[1][page, 0].astype(np.float64) * p.scales[1][page, 0].astype(np.float64)[:, None] for page in p.tables[r, :2])
        o, tol = (a + b) / 2, 38 * 2.0 ** -24 * (np.abs(a) + np.abs(b)) / 2
        for j in (2 * r, 2 * r + 1):
            assert np.all(np.abs(out[j] - o) <= tol), (j, float(np.max(np.abs(out[j] - o) / np.maximum(tol, 2.0 ** -60))))
            assert np.all(np.abs(lse[j] - np.log(32)) <= 42 * 2.0 ** -24), (j, lse[j] - np.log(32))
            worst = max(worst, float(np.max(np.abs(out[j] - o) / np.maximum(tol, 2.0 ** -60))))
    print(f"prompts over two blocks: at most {worst:.2f} of the bound", flush=True)


def test_equal_prompts_give_equal_bits(qmm):
    """A tile to a workgroup, and workgroups that share tiles: the same bits call after call, on
    whatever the workspace holds."""
    for held, new, heads, kv_heads, dim, q_t, c_t, out_t in (([0], [211], 64, 8, 128, BF16, I8, BF16), ([0], [1500], 16, 2, 128, BF16, I8, BF16),
                                                             ([900, 300, 30], [300, 120, 5], 32, 8, 64, F16, F16, F32)):
        c = prompt.Case(qmm, held, new, heads, kv_heads, dim, q_t, c_t, seed=dim)
        attn = qmm.PromptAttention(heads, kv_heads, dim, q_t, out_t)
        first = c.run(qmm, out_t, attn=attn)
        for fill in (0, 0x7F, 0xFF, 0x3C):
            attn.work.fill(fill)
            got = c.run(qmm, out_t, attn=attn)
            assert np.array_equal(got[0], first[0]) and np.array_equal(got[1].view(np.uint32), first[1].view(np.uint32)), fill
