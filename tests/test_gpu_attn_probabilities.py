"""Decode attention where its 16-bit parts of the probabilities are put to the test: a key far
above the others whose value is 0, so that the output is made of small probabilities alone,
and scores without an error of their own, so that the parts' is what is left.

A key has one nonzero dimension, q has 1 there and the scale is 1: a score is an element of
the cache, its product exact.  In powers of two, x = score * log2(e), the kernel rounds the
scale and the product (2^-24 of |x| each), the difference to the base (2^-24 of it, at most
|x| + |top| + 15) and the exponential (2^-22 of p): `spread` of p, relative.  Parts hold 2^-22 (fp16) or 2^-24
(bf16) of p.  With values that are not negative every term of numerator and denominator is
off by that much at most, and their sums in 32 bits by 2^-24 for each 32 keys and join."""
import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8
from test_gpu_attn_decode import Case


def bound(scores, out, q_t, n):
    """How far the output [heads, dim] of scores [heads, n] may be off, worst case, and the log
    of the sum (base, exponent and logarithm are added in 32 bits and multiplied)."""
    x = np.abs(scores).max() * 1.4427
    spread = np.log(2) * (2 * x + (2 * x + 15)) * 2.0 ** -24 + 2.0 ** -22
    part, sums = 2.0 ** -22 if q_t == F16 else 2.0 ** -24, (n / 32 + 64) * 2.0 ** -24
    return (2 * spread + part + sums) * np.abs(out) + 2.0 ** -120, spread + sums + (x + 15) * 2.0 ** -22


def scored(qmm, lens, heads, kv, dim, q_t, c_t, scores_of, values_of, **kw):
    """A Case whose scores are scores_of(request, key head, keys), values values_of alike."""
    c = Case(qmm, lens, heads, kv, dim, q_t, c_t, **kw)
    at = [(7 * h + 3) % dim for h in range(kv)]
    q = np.zeros((len(lens), heads, dim))
    for h in range(heads):
        q[:, h, at[h // (heads // kv)]] = 1.0
    c.qb = ref.encode(q, q_t)
    c.q = ref.decode(c.qb, q_t)
    for r, n in enumerate(lens):
        pg, off = c.tables[r][np.arange(n) // c.page], np.arange(n) % c.page
        k, v = np.zeros((n, kv, dim)), np.zeros((n, kv, dim))
        for h in range(kv):
            k[:, h, at[h]] = scores_of(r, h, n) / c.k_scale
            v[:, h] = values_of(r, h, n) / c.v_scale
        kb, vb = ref.encode(k, c_t), ref.encode(v, c_t)
        c.kb[pg, off], c.vb[pg, off] = kb, vb
        c.keys[r], c.values[r] = ref.decode(kb, c_t) * c.k_scale, ref.decode(vb, c_t) * c.v_scale
    c.upload(qmm)
    return c


def check(c, got):
    out = ref.decode(got[0], F32)
    group = c.heads // c.kv
    for r, n in enumerate(c.lens):
        o, l, _, _ = ref.attention(c.q[r], c.keys[r], c.values[r], 1.0)
        s = np.stack([c.keys[r][:, h // group] @ c.q[r, h] for h in range(c.heads)])
        tol, l_tol = bound(s, o, c.q_t, n)
        assert np.all(np.abs(out[r] - o) <= tol), (r, n, float(np.nanmax(np.abs(out[r] - o) / tol)), float(np.nanmax(np.abs(out[r] - o) / o)))
        assert np.all(np.abs(got[1][r] - l) <= l_tol), (r, n, float(np.abs(got[1][r] - l).max() / l_tol))


@pytest.mark.gpu
@pytest.mark.parametrize("nats", [8, 12, 16, 17.2, 20, 25, 35])
@pytest.mark.parametrize("q_t,c_t,dim", [(F16, F16, 64), (F16, F16, 96), (F16, F16, 128), (F16, F16, 192), (F16, F16, 256), (F16, F8, 64),
                                         (F16, F8, 128), (F16, F8, 256), (BF16, BF16, 128), (BF16, F8, 96)])
def test_first_key_draws_the_weight(qmm, q_t, c_t, dim, nats):
    """One key `nats` above the rest, which are equal or within +-0.5, its value 0; first,
    amidst and last; rows taken whole and cut."""
    if c_t == F8 and nats > 25:
        pytest.skip("past e4m3's largest")
    for lens, place in (([300, 33, 1025], 0), ([5000, 700], 0), ([5000, 40, 700], None), ([4097], -1)):
        rng = np.random.default_rng(int(nats * 10) + dim)

        def scores(r, h, n):
            s = rng.uniform(-0.5, 0.5, n) if h else np.zeros(n)
            s[n // 2 if place is None else place] = nats
            return s

        def values(r, h, n):
            v = np.abs(rng.standard_normal((n, dim))) + 0.1
            v[n // 2 if place is None else place] = 0
            return v
        c = scored(qmm, lens, 8, 2, dim, q_t, c_t, scores, values, seed=dim)
        check(c, c.run(qmm, scale=1.0))


def _two_keys():
    """Scores 0 and -1 .. 0, of values 0 and 1."""
    return np.random.default_rng(3).uniform(-1, 0, 96)


@pytest.mark.gpu
@pytest.mark.parametrize("q_t,c_t", [(BF16, BF16), (F16, F16), (BF16, F8), (F16, F8)])
def test_parts_hold_the_probabilities(qmm, q_t, c_t):
    """Two keys, the second's probability is the output's numerator."""
    low = _two_keys()
    c = scored(qmm, [2] * 96, 4, 4, 64, q_t, c_t, lambda r, h, n: np.array([0, low[r] * (1 + h / 4)]),
               lambda r, h, n: np.array([[0.0], [3.0]]) * np.ones((2, 64)), seed=1)
    check(c, c.run(qmm, scale=1.0))


def test_bound_tells_the_parts_apart():
    """One part fewer than the kernel has is past the bound of those two keys."""
    for q_t, parts in ((BF16, 3), (F16, 2)):
        s = ref.decode(ref.encode(_two_keys(), q_t), q_t)
        p = np.exp(s)
        worst = {}
        for n in (parts, parts - 1):
            held, left = np.zeros_like(p), p
            for _ in range(n):
                h = ref.decode(ref.encode(left, q_t), q_t)
                held, left = held + h, left - h
            o, got = p / (1 + p), held / (1 + p)
            worst[n] = max(abs(g - w) / bound(np.array([[0.0, x]]), np.array([[w]]), q_t, 2)[0][0, 0] for g, w, x in zip(got, o, s))
        assert worst[parts] <= 0.25 and worst[parts - 1] > 1, worst


@pytest.mark.gpu
@pytest.mark.parametrize("size", [5.0, 5e4, 5e6, 1e7, 1.3e8, 2e9])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_of_any_size(qmm, size, sign):
    """Equal scores up to where a step of fp32 is far above one: the mean of the values, to the
    parts and the sums."""
    n = 200
    for q_t in (F16, BF16):
        rng = np.random.default_rng(int(size) % 1000)
        v = np.abs(rng.standard_normal((n, 64))) + 0.1
        c = scored(qmm, [n], 2, 1, 64, q_t, q_t, lambda r, h, m: np.full(m, 1.0), lambda r, h, m: v, seed=2)
        out = ref.decode(c.run(qmm, scale=sign * size)[0], F32)
        want = c.values[0][:, 0].mean(0)
        assert np.all(np.abs(out[0] - want) <= (2.0 ** -22 + (n / 32 + 64) * 2.0 ** -24) * want)


@pytest.mark.gpu
@pytest.mark.parametrize("q_t,c_t,bits", [(BF16, BF16, 0x7F80), (BF16, BF16, 0xFF80), (BF16, BF16, 0x7FC0), (F16, F16, 0x7C00), (F16, F16, 0x7E00),
                                          (F16, F8, 0x7F), (BF16, F8, 0xFF)])
def test_values_without_a_number(qmm, q_t, c_t, bits):
    """An infinite value makes its dimension infinite or NaN for the heads that read it, NaN makes it
    NaN, and nothing else: other dimensions, key heads and rows are as without it."""
    for lens in ([300, 40], [5000, 300]):
        c = Case(qmm, lens, 8, 2, 64, q_t, c_t, seed=21)
        want = c.run(qmm)
        c.vb[c.tables[0, 2], 5, 1, 37] = bits
        c.upload(qmm)
        got = c.run(qmm)
        same = np.ones(got[0].shape, bool)
        same[0, 4:, 37] = False
        assert np.array_equal(got[0][same], want[0][same]) and np.array_equal(got[1], want[1])
        hit = ref.decode(got[0], F32)[~same]
        assert not np.isfinite(hit).any() and (np.isinf(ref.decode(np.array([bits], ref.BITS[c_t]), c_t)[0]) or np.isnan(hit).all())
