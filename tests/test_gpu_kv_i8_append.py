"""The quantising cache write on the GPU.  v is not turned, so its codes and scales have to be
those of the header's formulas in 32 bits, bit for bit; k is turned in 32 bits, an error of at
most 2^-21 (|a| + |b|) of a pair (a, b) (sine and cosine within 2^-23, a product and a sum), so
its scales are held to 2^-20 and its codes to half a step more than that error's."""
import numpy as np
import pytest

import attn_ref as ref
import kv_i8_ref as kv
from attn_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu
I8 = kv.I8


class Step:
    """One call: `held` tokens of each request, `new` more of each (slots by the requests' tables, or
    given), into a cache whose blocks hold what `held` says."""

    def __init__(self, qmm, held, new, heads=4, kv_heads=2, dim=64, block=16, page=16, layout="token", in_t=F32, q_t=BF16, axes=1,
                 adjacent=False, rot=None, scale=1.0, seed=0, size=1.0, slots=None, extra=3):
        self.c = c = kv.Paged(qmm, [h + n for h, n in zip(held, new)], kv_heads, dim, I8, page, block, layout, seed, extra=extra)
        rng, self.dims = c.rng, (heads, kv_heads, dim)
        # scales that new elements of about `size` sometimes outgrow
        for s in c.scales:
            s[:] = (rng.uniform(0.5, 1.5, s.shape) * size * 3 / 127).astype(np.float32)
        c.upload(qmm)
        rows = [r for r, n in enumerate(new) for _ in range(n)]
        at = [h + i for h, n in zip(held, new) for i in range(n)]
        self.slots = [int(c.tables[r, p // page]) * page + p % page for r, p in zip(rows, at)] if slots is None else list(slots)
        n = len(self.slots)
        self.x = [ref.encode(rng.standard_normal((n, h, dim)) * size, in_t) for h in (heads, kv_heads, kv_heads)]
        self.in_t, self.q_t, self.adjacent, self.scale = in_t, q_t, adjacent, scale
        pairs = (rot or dim) // 2
        self.freq, self.axis = qmm.rope_frequencies(pairs), [i % axes for i in range(pairs)]
        self.pos = rng.integers(0, 100000, (axes, n)).astype(np.int32)

    def run(self, qmm, stream=None):
        c, (heads, kv_heads, dim), n = self.c, self.dims, len(self.slots)
        print(f"append_i8 tokens={n} heads={heads}/{kv_heads} dim={dim} block={c.block} page={c.page} {c.layout} in={self.in_t}", flush=True)
        rope = qmm.Rope(self.freq, axes=self.axis, n_axes=len(self.pos), pairing="adjacent" if self.adjacent else "halves", scale=self.scale)
        d = [qmm.DeviceBuffer.from_numpy(x) for x in self.x]
        dq = qmm.DeviceBuffer(max(n * heads * dim * 2, 16))
        dpos, dslots = qmm.DeviceBuffer.from_numpy(self.pos), qmm.DeviceBuffer.from_numpy(np.array(self.slots, np.int32))
        rope.append(c.cache, *d, self.in_t, dq, self.q_t, dpos, dslots, n, heads, stream=stream)
        return dq.download(np.uint16, (n, heads, dim), stream), c.download(stream)

    def check(self, q, after, runs=None, errors=True):
        c, n = self.c, len(self.slots)
        xs = [ref.decode(x, self.in_t) for x in self.x]
        turned = [ref.rope(x, self.pos, self.freq, self.axis, self.adjacent, self.scale) for x in xs[:2]]
        # of a pair, at most 2^-21 of |a| + |b|, which is sqrt(2) of the pair's length at most
        slack = [2.0 ** -20 * abs(self.scale) * np.abs(x).max(-1, keepdims=True) for x in xs[:2]]
        got = ref.decode(q, self.q_t)
        assert np.all(np.abs(got - turned[0]) <= ref.ROUND[self.q_t] * np.abs(turned[0]) + 2 * slack[0] + ref.TINY[self.q_t])
        runs = kv.runs(self.slots, c.block, c.n_pages * c.page) if runs is None else runs
        for i, x in enumerate((turned[1], xs[2])):
            before_c, before_s = c.bits[i], c.scales[i]
            after_c, after_s = after[i]
            want_c, want_s = before_c.copy(), before_s.copy()
            for first, count in runs:
                page, off = divmod(self.slots[first], c.page)
                b, held = off // c.block, off % c.block
                lo = off - held
                for h in range(self.dims[1]):
                    new = x[first:first + count, h]
                    most, old = np.abs(new).max(), before_s[page, b, h]
                    s = kv.new_scale(np.float32(most) if np.isfinite(new).all() else np.nan, held, old)
                    mine = after_s[page, b, h]
                    want_s[page, b, h] = mine
                    if not np.isfinite(s) or i == 1:
                        assert np.array_equal(mine, s, equal_nan=True), (i, first, h, mine, s)
                    else:
                        assert abs(float(mine) - float(s)) <= 2.0 ** -20 * float(s) + slack[1][first:first + count, h].max() / 127, (first, h, mine, s)
                    codes = after_c[page, off:off + count, h]
                    want_c[page, off:off + count, h] = codes
                    if not np.isfinite(mine):
                        continue
                    if mine != old and held:
                        want_c[page, lo:off, h] = kv.rescaled(before_c[page, lo:off, h], old, mine)
                    if i == 1:
                        assert np.array_equal(codes, kv.codes_of(new, mine)), (first, h)
                    else:
                        off_by = np.abs(codes - np.clip(new / float(mine), -127, 127))
                        assert np.all(off_by <= 0.5 + 2.0 ** -15 + 2 * slack[1][first:first + count, h] / float(mine)), (first, h, off_by.max())
            assert np.array_equal(after_c, want_c), ("codes", i, np.argwhere(after_c != want_c)[:5])
            assert np.array_equal(after_s, want_s, equal_nan=True), ("scales", i)
            c.bits[i], c.scales[i] = after_c, after_s


HELD, NEW = [0, 1, 15, 16, 17, 31, 40, 5], [1, 1, 1, 1, 16, 40, 3, 0]


@pytest.mark.parametrize("block,page", [(8, 8), (8, 24), (16, 16), (16, 64), (32, 32), (32, 160)])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_blocks_and_layouts(qmm, block, page, layout):
    s = Step(qmm, HELD, NEW, block=block, page=page, layout=layout, seed=block + page)
    s.check(*s.run(qmm))


@pytest.mark.parametrize("dim,rot,block", [(16, 8, 8), (48, 16, 16), (64, 64, 32), (96, 96, 16), (128, 64, 32), (192, 192, 16), (256, 256, 32),
                                           (256, 128, 8)])
@pytest.mark.parametrize("in_t,adjacent", [(F32, False), (F16, True), (BF16, False)])
def test_dims_and_types(qmm, dim, rot, block, in_t, adjacent):
    s = Step(qmm, HELD, NEW, dim=dim, rot=rot, block=block, page=32, in_t=in_t, adjacent=adjacent, axes=3 if rot > 8 else 1, scale=1.25,
             q_t=F16, seed=dim + rot)
    s.check(*s.run(qmm))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (64, 8), (5, 5), (32, 32)])
def test_heads(qmm, heads, kv_heads):
    s = Step(qmm, [3, 30], [2, 35], heads, kv_heads, 128, seed=heads)
    s.check(*s.run(qmm))


def test_single_tokens_and_long_prompts(qmm):
    """Many requests, and so many tokens that heads share a workgroup and loads stream."""
    rng = np.random.default_rng(3)
    s = Step(qmm, [int(n) for n in rng.integers(0, 90, 300)], [1] * 300, 16, 8, 128, block=16, page=32, seed=1)
    s.check(*s.run(qmm))
    for block in (8, 32):
        s = Step(qmm, [7, 11], [3001, 1500], 4, 4, 64, block=block, page=64, seed=block)
        s.check(*s.run(qmm))
    s = Step(qmm, [5], [1100], 2, 32, 64, block=16, page=16, layout="head", in_t=BF16, seed=4)
    s.check(*s.run(qmm))


def test_a_block_that_fills_token_by_token(qmm):
    """Elements that grow: the scale grows by a quarter at least, held codes are rounded again, and
    the sum of all roundings stays below 2.5 steps of the last scale."""
    s = Step(qmm, [0], [16], 2, 2, 64, seed=5)
    c, page = s.c, int(s.c.tables[0, 0])
    want, scales = [], []
    all_x, all_pos = s.x, s.pos
    for t in range(16):
        grow = 1.13 ** t
        s.slots = [page * 16 + t]
        s.x = [ref.encode(ref.decode(x[t:t + 1], F32) * grow, F32) for x in all_x]
        s.pos = all_pos[:, t:t + 1]
        want.append(ref.decode(s.x[2], F32)[0])
        s.check(*s.run(qmm))
        scales.append(c.scales[1][page, 0].copy())
    scales = np.array(scales)
    grown = scales[1:] / scales[:-1]
    assert np.all((grown == 1) | (grown >= 1.2499)) and (grown > 1).any()
    back = c.bits[1][page].astype(np.float64) * scales[-1][:, None].astype(np.float64)
    assert np.all(np.abs(back - np.array(want)) <= 2.5 * scales[-1][:, None])


def test_slots_that_are_not_taken(qmm):
    """Refused tokens and slots past the cache write q alone, and break a run."""
    s = Step(qmm, [0], [64], 2, 2, 64, seed=6)
    c = s.c
    n = c.n_pages * c.page
    p = [int(x) * 16 for x in c.tables[0, :4]]
    s.slots = [p[0] + 3, p[0] + 4, -1, p[0] + 7, n, n + 5, 2 ** 31 - 1, -2 ** 31, p[1], p[1] + 1, p[1] + 2, -7, p[2] + 15, p[3], p[3] + 1, -1]
    s.x, s.pos = [x[:16] for x in s.x], s.pos[:, :16]
    # two runs of one block in one call: what it holds afterwards is not said; the other blocks are
    q, after = s.run(qmm)
    for i in range(2):
        for a, b in ((after[i][0], c.bits[i]), (after[i][1], c.scales[i])):
            b[p[0] // 16] = a[p[0] // 16]
    s.check(q, after, runs=[r for r in kv.runs(s.slots, 16, n) if s.slots[r[0]] // 16 != p[0] // 16])


def test_zeros_and_extremes(qmm):
    """A block of zeros, of the least and of the largest numbers; no element of a block is above its
    scale's 127."""
    s = Step(qmm, [0, 0, 0, 4, 4], [3, 3, 3, 1, 1], 2, 2, 64, seed=7)
    x = [ref.decode(a, F32) for a in s.x]
    for a in x[1:]:
        a[0:3] = 0
        a[3:6] *= 1e-30
        a[6:9] *= 2e37
        a[9:10] *= 1e9
        a[10:11] = 0
    s.x = [ref.encode(a, F32) for a in x]
    q, after = s.run(qmm)
    s.check(q, after)
    c = s.c
    first = int(c.tables[0, 0])
    assert np.all(after[0][1][first] == 2.0 ** -40) and not after[0][0][first, :3].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_without_a_number(qmm, bad):
    """They make their block's scale NaN, of their head alone, until it is started anew."""
    s = Step(qmm, [2, 0, 20], [1, 20, 2], 2, 2, 64, seed=8)
    x = [ref.decode(a, F32) for a in s.x]
    x[1][0, 1, 5] = bad       # k of request 0, head 1
    x[2][1 + 17, 0, 63] = bad  # v of request 1's second block
    s.x = [ref.encode(a, F32) for a in x]
    _, after = s.run(qmm)
    c = s.c
    p0, p1 = int(c.tables[0, 0]), int(c.tables[1, 1])
    assert np.isnan(after[0][1][p0, 0, 1]) and np.isfinite(after[0][1][p0, 0, 0]) and np.isfinite(after[1][1][p0]).all()
    assert np.isnan(after[1][1][p1, 0, 0]) and np.isfinite(after[1][1][p1, 0, 1]) and np.isfinite(after[0][1][p1]).all()
    # a later token leaves it so, a first token does not
    for i in range(2):
        c.bits[i], c.scales[i] = after[i]
    s.slots, s.pos = [p0 * 16 + 3, p1 * 16], s.pos[:, :2]
    s.x = [ref.encode(ref.decode(a, F32)[1:3], F32) for a in s.x]
    _, after = s.run(qmm)
    assert np.isnan(after[0][1][p0, 0, 1]) and np.isfinite(after[1][1][p1]).all()


def test_strided_inputs_and_streams(qmm):
    """q, k and v as slices of one projection, on another stream, twice: the second call finds
    scales that are large enough and changes nothing."""
    s = Step(qmm, [9, 0], [4, 18], 4, 2, 64, seed=9)
    c, n = s.c, 22
    row = (4 + 2 + 2) * 64 + 8
    wide = np.full((n, row), np.nan, np.float32)
    at = 0
    for x, h in zip(s.x, (4, 2, 2)):
        wide[:, at:at + h * 64] = ref.decode(x, F32).reshape(n, -1)
        at += h * 64
    d, st = qmm.DeviceBuffer.from_numpy(wide), qmm.Stream()
    part = [kv.at_page(d, off * 4, d.nbytes - off * 4) for off in (0, 256, 384)]
    rope, dq = qmm.Rope(s.freq, axes=s.axis), qmm.DeviceBuffer(n * 256 * 2)
    dpos, dslots = qmm.DeviceBuffer.from_numpy(s.pos), qmm.DeviceBuffer.from_numpy(np.array(s.slots, np.int32))
    results = []
    for _ in range(2):
        print("append_i8 strided", flush=True)
        rope.append(c.cache, *part, F32, dq, BF16, dpos, dslots, n, 4, stream=st.handle, q_stride=row, k_stride=row, v_stride=row)
        results.append((dq.download(np.uint16, (n, 4, 64), st.handle), c.download(st.handle)))
    for (a, b), (e, f) in zip(results[0][1], results[1][1]):
        assert np.array_equal(a, e) and np.array_equal(b, f, equal_nan=True)
    s.check(*results[0])


def test_offsets_past_32_bits(qmm):
    """Slots more than 4 GiB into keys and values, and scales' places past 2^31."""
    page, kv_heads, dim = 256, 8, 128
    per_page = page * kv_heads * dim
    n_pages = (9 << 29) // per_page + 1
    s = Step(qmm, [0, 300], [40, 1], 8, kv_heads, dim, page=page, block=32, seed=10)
    c = s.c
    d = [qmm.DeviceBuffer(n_pages * per_page) for _ in range(2)]
    ds = [qmm.DeviceBuffer(n_pages * 8 * kv_heads * 4) for _ in range(2)]
    shift = n_pages - c.n_pages
    for i in range(2):
        for buf, src, each in ((d[i], c.bits[i], per_page), (ds[i], c.scales[i], 8 * kv_heads * 4)):
            qmm.stream_copy(kv.at_page(buf, shift * each, src.nbytes), qmm.DeviceBuffer.from_numpy(src), src.nbytes)
    whole = qmm.KVCache(d[0], d[1], I8, n_pages, page, kv_heads, dim, block=32, d_k_scales=ds[0], d_v_scales=ds[1])
    n = len(s.slots)
    rope, dq = qmm.Rope(s.freq, axes=s.axis), qmm.DeviceBuffer(n * 8 * dim * 2)
    dslots = qmm.DeviceBuffer.from_numpy(np.array([x + shift * page for x in s.slots], np.int32))
    print(f"append_i8 into {n_pages * per_page} bytes", flush=True)
    rope.append(whole, *[qmm.DeviceBuffer.from_numpy(x) for x in s.x], F32, dq, BF16, qmm.DeviceBuffer.from_numpy(s.pos), dslots, n, 8)
    after = []
    for i in range(2):
        both = []
        for buf, like, each in ((d[i], c.bits[i], per_page), (ds[i], c.scales[i], 8 * kv_heads * 4)):
            out = qmm.DeviceBuffer(like.nbytes)
            qmm.stream_copy(out, kv.at_page(buf, shift * each, like.nbytes), like.nbytes)
            both.append(out.download(like.dtype, like.shape))
        after.append(tuple(both))
    s.check(dq.download(np.uint16, (n, 8, dim)), after)


def test_graph_replays(qmm):
    """A captured call, replayed with other tokens in its buffers, is the eager call."""
    from openmini_qmm.hip_runtime import Graph
    s, e = (Step(qmm, [9, 30], [1, 1], 4, 2, 64, seed=11) for _ in range(2))
    st = qmm.Stream()
    rope = qmm.Rope(s.freq, axes=s.axis)
    d = [qmm.DeviceBuffer.from_numpy(x) for x in s.x]
    dq, dpos, dslots = qmm.DeviceBuffer(2 * 4 * 64 * 2), qmm.DeviceBuffer.from_numpy(s.pos), qmm.DeviceBuffer.from_numpy(np.array(s.slots, np.int32))
    g = Graph(st.handle, lambda h: rope.append(s.c.cache, *d, F32, dq, BF16, dpos, dslots, 2, 4, stream=h))
    rng = np.random.default_rng(0)
    for rep in range(4):
        x = [ref.encode(rng.standard_normal(a.shape) * 1.5 ** rep, F32) for a in s.x]
        for buf, a in zip(d, x):
            buf.upload(a, st.handle)
        print(f"append_i8 graph replay {rep}", flush=True)
        g.launch(st.handle)
        st.synchronize()
        s.x = e.x = x
        got = dq.download(np.uint16, (2, 4, 64)), s.c.download()
        s.check(*got)
        eager = e.run(qmm)
        assert np.array_equal(eager[0], got[0])
        for (a, b), (f, h) in zip(eager[1], got[1]):
            assert np.array_equal(a, f) and np.array_equal(b, h, equal_nan=True)
        e.check(*eager)
        slots = [x + 1 for x in s.slots]
        s.slots = e.slots = [x if x % 16 else y for x, y in zip(slots, s.slots)]
        dslots.upload(np.array(s.slots, np.int32), st.handle)


def test_refusals(qmm):
    s = Step(qmm, [0], [1], 2, 2, 64)
    rope = qmm.Rope(s.freq)
    d = qmm.DeviceBuffer(1 << 16)
    with pytest.raises(qmm.InvalidInput):
        rope.append(s.c.cache, kv.at_page(d, 0, 8), d, d, F32, d, BF16, d, d, 1, 2)
    for dim in (8, 40):  # rows of a cache are multiples of 16 bytes
        odd = kv.Paged(qmm, [8], 2, dim, I8)
        with pytest.raises(qmm.QmmError, match="multiple of 16 bytes"):
            rope.append(odd.cache, d, d, d, F32, qmm.DeviceBuffer(1 << 12), BF16, d, d, 1, 2)
    wide = kv.Paged(qmm, [8], 1, 512, I8)
    with pytest.raises(qmm.QmmError, match="at most 256"):
        rope.append(wide.cache, d, d, d, F32, qmm.DeviceBuffer(1 << 12), BF16, d, d, 1, 1)
    big = qmm._native.RopeAppendArgs(d.ptr, d.ptr, d.ptr, 128, 128, 128, qmm.DeviceBuffer(64).ptr, 128, F32, BF16, 1 << 28, 2, d.ptr, 1 << 28, d.ptr)
    assert qmm.lib().openmini_rope_append_i8(rope.handle, s.c.cache.desc, s.c.cache.scales, big, None) == qmm._native.ERR_INVALID_PARAM
    rope.append(s.c.cache, d, d, d, F32, qmm.DeviceBuffer(64), BF16, d, d, 0, 2)  # no tokens
