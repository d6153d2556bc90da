"""Rotary positions and the cache write on the GPU, against 64 bits.  An angle is exact to
2^-31 of a turn and its sine to 2e-9 and fp32 rounding, so a turned element is within
2^-21 (|a| + |b|) |scale| of its pair's exact turn, then rounded to the output's type."""
import ctypes

import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8

pytestmark = pytest.mark.gpu


def _freq(pairs):
    return [10000.0 ** (-i / pairs) for i in range(pairs)]


def _inputs(rng, shape, t):
    bits = ref.encode(rng.standard_normal(shape), t)
    return bits, ref.decode(bits, t)


def _size(x, pairs, adjacent):
    """|a| + |b| of each element's pair (its own size where it passes through)."""
    a = np.abs(x)
    out = np.array(a)
    i, j = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    out[..., i] = out[..., j] = a[..., i] + a[..., j]
    return out


def _close(got, want, size, t, scale=1.0, what=""):
    tol = 2.0 ** -21 * size * max(abs(scale), 1.0)
    tol = tol + ref.ROUND[t] * (np.abs(want) + tol) + ref.TINY[t]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / tol)))


@pytest.mark.parametrize("xt,yt", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (F16, F32), (BF16, F16)])
@pytest.mark.parametrize("tokens,heads,dim,pairs,axes,adjacent", [
    (1, 1, 8, 4, 1, False), (1, 32, 128, 64, 1, False), (3, 5, 96, 24, 3, True), (17, 3, 64, 32, 2, False),
    (301, 16, 128, 64, 3, True), (70, 1, 256, 128, 8, False), (9, 40, 40, 12, 1, True), (5, 2, 512, 128, 3, False)])
def test_apply(qmm, xt, yt, tokens, heads, dim, pairs, axes, adjacent):
    rng = np.random.default_rng(tokens * 7 + heads)
    print(f"rope {tokens} x {heads} x {dim}, {pairs} pairs, {axes} axes, adjacent={adjacent} {xt}->{yt}", flush=True)
    bits, x = _inputs(rng, (tokens, heads, dim), xt)
    pos = rng.integers(-50, 40000, (axes, tokens)).astype(np.int32)
    axis = [int(a) for a in rng.integers(0, axes, pairs)]
    axis[0] = axes - 1
    scale = 1.0 if heads % 2 else 1.1386
    r = qmm.Rope(_freq(pairs), axes=axis, n_axes=axes, pairing="adjacent" if adjacent else "halves", scale=scale)
    dx, dp = qmm.DeviceBuffer.from_numpy(bits), qmm.DeviceBuffer.from_numpy(pos)
    for inverse in (False, True):
        dy = qmm.DeviceBuffer(x.size * ref.SIZE[yt])
        r.apply(dx, xt, dy, yt, dp, tokens, heads, dim, inverse=inverse)
        got = ref.decode(dy.download(ref.BITS[yt], x.shape), yt)
        want = ref.rope(x, pos, _freq(pairs), axis, adjacent, scale, inverse)
        _close(got, want, _size(x, pairs, adjacent), yt, scale, f"inverse={inverse}")
        if 2 * pairs < dim and xt == yt:  # what is not turned passes through, bit for bit
            assert np.array_equal(dy.download(ref.BITS[yt], x.shape)[..., 2 * pairs:], bits[..., 2 * pairs:])


def test_far_positions(qmm):
    """Positions to the ends of int32: the angle's reduction is exact."""
    pos = np.array([[0, 1, -1, 100000, 1 << 24, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31]], np.int32)
    rng = np.random.default_rng(3)
    bits, x = _inputs(rng, (8, 2, 64), F32)
    r = qmm.Rope(_freq(32))
    dy = qmm.DeviceBuffer(x.size * 4)
    print("rope far positions", flush=True)
    r.apply(qmm.DeviceBuffer.from_numpy(bits), F32, dy, F32, qmm.DeviceBuffer.from_numpy(pos), 8, 2, 64)
    # a frequency is kept to 2^-65 of a turn, and its division by 2 pi in 80 bits is as exact
    # as that: 2^31 positions later 2^-33 of a turn, within the bound's 2^-21
    _close(dy.download(np.float32, x.shape).astype(np.float64), ref.rope(x, pos, _freq(32), [0] * 32), _size(x, 32, False), F32)


def test_strides_in_place_and_stream(qmm):
    rng = np.random.default_rng(4)
    tokens, heads, dim, stride = 37, 4, 64, 4 * 64 + 24
    bits, x = _inputs(rng, (tokens, stride), F32)
    x3 = x[:, :heads * dim].reshape(tokens, heads, dim)
    pos = np.zeros((3, 50), np.int32)
    pos[:, :tokens] = rng.integers(0, 500, (3, tokens))
    axis = [i % 3 for i in range(32)]
    s = qmm.Stream()
    r = qmm.Rope(_freq(32), axes=axis)
    d = qmm.DeviceBuffer.from_numpy(bits)
    print("rope in place, strided", flush=True)
    r.apply(d, F32, d, F32, qmm.DeviceBuffer.from_numpy(pos), tokens, heads, dim, x_stride=stride, y_stride=stride, position_stride=50,
            stream=s.handle)
    got = d.download(np.float32, bits.shape, s.handle)
    _close(got[:, :heads * dim].reshape(x3.shape).astype(np.float64), ref.rope(x3, pos[:, :tokens], _freq(32), axis), _size(x3, 32, False), F32)
    assert np.array_equal(got[:, heads * dim:].view(np.uint32), bits[:, heads * dim:])


def test_gradient(qmm):
    """inverse is the gradient: by the formula (its transpose) and by differences."""
    rng = np.random.default_rng(6)
    shape, pairs = (3, 2, 32), 12
    pos = rng.integers(0, 3000, (1, 3)).astype(np.int32)
    r = qmm.Rope(_freq(pairs), pairing="adjacent", scale=0.7)
    dp = qmm.DeviceBuffer.from_numpy(pos)

    def turn(v, inverse=False):
        dy = qmm.DeviceBuffer(v.size * 4)
        r.apply(qmm.DeviceBuffer.from_numpy(v.astype(np.float32)), F32, dy, F32, dp, *shape, inverse=inverse)
        return dy.download(np.float32, shape).astype(np.float64)

    x, g = (rng.standard_normal(shape).astype(np.float32).astype(np.float64) for _ in range(2))
    grad = turn(g, inverse=True)
    want = ref.rope(g, pos, _freq(pairs), [0] * pairs, True, 0.7, True)
    _close(grad, want, _size(g, pairs, True), F32)
    # L = sum g . y is linear in x: a step of 1 gives its derivative but for roundings
    base = np.sum(g * turn(x))
    for at in [(0, 0, 0), (1, 1, 13), (2, 0, 23), (2, 1, 24), (0, 1, 31)]:
        e = np.zeros(shape)
        e[at] = 1.0
        assert abs((np.sum(g * turn(x + e)) - base) - grad[at]) < 1e-4, at


def test_refusals(qmm):
    from openmini_qmm import QmmError
    r = qmm.Rope(_freq(32), axes=[i % 2 for i in range(32)])
    d = qmm.DeviceBuffer(1 << 16)
    for kw, word in ((dict(head_dim=56), "do not fit"), (dict(head_dim=60), "multiple of 8"), (dict(heads=0), "heads"),
                     (dict(x_dtype=F8), "not taken"), (dict(y_dtype=F8), "not taken"), (dict(x_stride=63), "x_stride"),
                     (dict(y_stride=66), "y_stride"), (dict(y_dtype=BF16), "in place"), (dict(position_stride=1), "position_stride")):
        a = dict(d_x=d, x_dtype=F32, d_y=d, y_dtype=F32, d_positions=d, tokens=2, heads=1, head_dim=64)
        a.update(kw)
        with pytest.raises((QmmError, qmm.InvalidInput), match=word):
            r.apply(**a)
    with pytest.raises(qmm.InvalidInput):
        r.apply(d, F32, d, F32, d, 2000, 1, 64)
    r.apply(d, F32, d, F32, d, 0, 1, 64)  # no tokens: nothing to do


def _append(qmm, rng, tokens, heads, kv, dim, pairs, axes, in_t, q_t, c_t, page, layout, slots, n_pages, fused=False, adjacent=False):
    print(f"append {tokens} x {heads}/{kv} x {dim} {in_t} -> q {q_t} cache {c_t} page {page} {layout}", flush=True)
    pos = rng.integers(0, 9000, (axes, tokens)).astype(np.int32)
    axis = [i % axes for i in range(pairs)]
    scale = 1.25
    r = qmm.Rope(_freq(pairs), axes=axis, n_axes=axes, scale=scale, pairing="adjacent" if adjacent else "halves")
    total = heads + 2 * kv
    bits, x = _inputs(rng, (tokens, total, dim), in_t)
    if c_t == F8:  # past the largest code, infinite and NaN values too
        x[0, heads + kv, :4] = [1e6, -1e6, np.inf, np.nan]
        bits = ref.encode(x, in_t)
        x = ref.decode(bits, in_t)
    parts = (slice(0, heads), slice(heads, heads + kv), slice(heads + kv, total))
    size = ref.SIZE[in_t]
    if fused:
        d = qmm.DeviceBuffer.from_numpy(bits)

        class At:
            def __init__(self, first):
                self.ptr = ctypes.c_void_p(d.ptr.value + first * dim * size)
                self.nbytes = d.nbytes - first * dim * size
        bufs = [At(p.start) for p in parts]
        strides = dict(q_stride=total * dim, k_stride=total * dim, v_stride=total * dim)
    else:
        bufs = [qmm.DeviceBuffer.from_numpy(np.ascontiguousarray(bits[:, p])) for p in parts]
        strides = {}
    shape = (n_pages, page, kv, dim) if layout == "token" else (n_pages, kv, page, dim)
    before = [rng.integers(0, 256, np.prod(shape) * ref.SIZE[c_t]).astype(np.uint8).view(ref.BITS[c_t]).reshape(shape) for _ in range(2)]
    dk, dv = (qmm.DeviceBuffer.from_numpy(b) for b in before)
    ks, vs = (0.25, 0.02) if c_t == F8 else (1.0, 1.0)
    cache = qmm.KVCache(dk, dv, c_t, n_pages, page, kv, dim, layout=layout, k_scale=ks, v_scale=vs)
    dq = qmm.DeviceBuffer(tokens * heads * dim * 2)
    r.append(cache, *bufs, in_t, dq, q_t, qmm.DeviceBuffer.from_numpy(pos), qmm.DeviceBuffer.from_numpy(slots.astype(np.int32)), tokens, heads,
             **strides)
    q, k, v = (x[:, p] for p in parts)
    turn = lambda t: ref.rope(t, pos, _freq(pairs), axis, adjacent, scale)  # noqa: E731
    _close(ref.decode(dq.download(ref.BITS[q_t], q.shape), q_t), turn(q), _size(q, pairs, adjacent), q_t, scale, "q")
    for name, new, sz, buf, old, sc in (("k", turn(k), _size(k, pairs, adjacent), dk, before[0], ks), ("v", v, np.abs(v) * 0, dv, before[1], vs)):
        got_bits = buf.download(ref.BITS[c_t], shape)
        by_token = got_bits if layout == "token" else got_bits.swapaxes(1, 2)
        untouched = np.ones((n_pages, page), bool)
        for j, s in enumerate(slots):
            if 0 <= s < n_pages * page:
                untouched[s // page, s % page] = False
                want, got = new[j] / sc, ref.decode(by_token[s // page, s % page], c_t)
                if c_t == F8:
                    nan = np.isnan(want)
                    assert np.array_equal(np.isnan(got), nan), name
                    want, got = np.where(nan, 0, np.clip(want, -448, 448)), np.where(nan, 0, got)
                tol = 2.0 ** -21 * np.where(np.isfinite(sz[j]), sz[j], 0) * scale / sc + 2.0 ** -23 * np.abs(want)
                tol = tol + ref.ROUND[c_t] * (np.abs(want) + tol) + ref.TINY[c_t]
                assert np.all(np.abs(got - want) <= tol), (name, j, float(np.max(np.abs(got - want) / tol)))
        old_by_token = old if layout == "token" else old.swapaxes(1, 2)
        assert np.array_equal(by_token[untouched], old_by_token[untouched]), name


@pytest.mark.parametrize("in_t,q_t,c_t", [(F32, BF16, BF16), (F32, F16, F16), (F32, BF16, F8), (BF16, BF16, BF16), (F16, F16, F8),
                                          (F32, F16, BF16)])
@pytest.mark.parametrize("tokens,heads,kv,dim,pairs,axes,page,layout,adjacent", [
    (1, 8, 1, 128, 64, 1, 16, "token", False), (1, 64, 8, 128, 64, 1, 16, "head", False), (5, 6, 2, 64, 32, 3, 8, "head", True),
    (33, 4, 4, 96, 24, 1, 17, "token", False), (300, 12, 3, 256, 128, 2, 64, "token", True)])
def test_append(qmm, in_t, q_t, c_t, tokens, heads, kv, dim, pairs, axes, page, layout, adjacent):
    rng = np.random.default_rng(tokens + heads + c_t)
    n_pages = tokens // page + 4
    slots = rng.permutation(n_pages * page)[:tokens]
    _append(qmm, rng, tokens, heads, kv, dim, pairs, axes, in_t, q_t, c_t, page, layout, slots, n_pages, adjacent=adjacent)


def test_append_slots_outside(qmm):
    """Negative slots and slots past the cache write nothing but q."""
    rng = np.random.default_rng(11)
    slots = np.array([-1, 63, 64, 5, -2 ** 31, 2 ** 31 - 1, 0])
    _append(qmm, rng, 7, 4, 2, 64, 32, 1, F32, BF16, BF16, 16, "token", slots, 4)


def test_append_fused_projection(qmm):
    """q, k and v as slices of one array."""
    rng = np.random.default_rng(12)
    _append(qmm, rng, 21, 8, 2, 128, 64, 3, F32, BF16, F8, 16, "head", rng.permutation(160)[:21], 10, fused=True)
    _append(qmm, rng, 21, 8, 2, 128, 64, 3, BF16, BF16, BF16, 16, "token", rng.permutation(160)[:21], 10, fused=True)


def test_append_refusals(qmm):
    from openmini_qmm import QmmError
    r, d = qmm.Rope(_freq(32)), qmm.DeviceBuffer(1 << 16)
    e = qmm.DeviceBuffer(1 << 16)
    c = qmm.KVCache(d, d, BF16, 4, 16, 2, 64)
    for kw, word in ((dict(in_dtype=F8), "not taken"), (dict(q_dtype=F32), "not taken"), (dict(q_heads=0), "heads"),
                     (dict(d_q_out=d), "one of the inputs"), (dict(k_stride=100), "k_stride")):
        a = dict(cache=c, d_q=d, d_k=d, d_v=d, in_dtype=F32, d_q_out=e, q_dtype=BF16, d_positions=d, d_slots=d, tokens=2, q_heads=4)
        a.update(kw)
        with pytest.raises((QmmError, qmm.InvalidInput), match=word):
            r.append(**a)
