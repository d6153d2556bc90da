"""Attention of single tokens over a paged cache on the GPU, against 64 bits, at the bounds
of attn_ref.attention_bounds.  Pages lie anywhere in the cache; what no row sees holds NaN."""
import ctypes

import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8

pytestmark = pytest.mark.gpu
NAN = {BF16: 0x7FC0, F16: 0x7E00, F8: 0x7F}


class Case:
    """Inputs of a call: `lens` keys of each request; rows[j] reads request reqs[j]."""

    def __init__(self, qmm, lens, heads, kv, dim, q_t=BF16, c_t=BF16, page=16, layout="token", reqs=None, row_lens=None, seed=0,
                 k_size=1.0, max_pages=None, window=0):
        rng = np.random.default_rng(seed)
        self.rng, self.heads, self.kv, self.dim, self.q_t, self.c_t, self.page, self.layout = rng, heads, kv, dim, q_t, c_t, page, layout
        self.lens, self.window = list(lens), window
        self.reqs = list(range(len(lens))) if reqs is None else list(reqs)
        self.row_lens = list(lens) if row_lens is None else list(row_lens)
        self.mapped = reqs is not None
        held = [-(-n // page) for n in lens]
        self.max_pages = max_pages or max(max(held), 1)
        self.n_pages = sum(held) + 3
        order = rng.permutation(self.n_pages).astype(np.int32)
        # entries past a request's pages: anything at all
        self.tables = rng.choice(np.array([-1, -2 ** 31, 2 ** 31 - 1, self.n_pages, 0], np.int32), (len(lens), self.max_pages))
        at = 0
        for r, h in enumerate(held):
            self.tables[r, :h] = order[at:at + h]
            at += h
        self.k_scale, self.v_scale = (0.0625, 0.3) if c_t == F8 else (1.0, 1.0)
        spread = 16.0 if c_t == F8 else 1.0
        shape = (self.n_pages, page, kv, dim)
        self.kb, self.vb = (np.full(shape, NAN[c_t], ref.BITS[c_t]) for _ in range(2))
        self.keys, self.values = [], []
        for r, n in enumerate(lens):
            if n == 0:
                self.keys.append(np.zeros((0, kv, dim)))
                self.values.append(np.zeros((0, kv, dim)))
                continue
            pg, off = self.tables[r][np.arange(n) // page], np.arange(n) % page
            lo = max(0, min((rl for q, rl in zip(self.reqs, self.row_lens) if q == r), default=n) - window) if window else 0
            for bits, out, size, sc in ((self.kb, self.keys, k_size * spread, self.k_scale), (self.vb, self.values, spread, self.v_scale)):
                b = ref.encode(rng.standard_normal((n, kv, dim)) * size, c_t)
                b[:lo // 8 * 8] = NAN[c_t]  # before every window: pages given back
                bits[pg, off] = b
                out.append(ref.decode(b, c_t) * sc)
        self.qb = ref.encode(rng.standard_normal((len(self.reqs), heads, dim)), q_t)
        self.q = ref.decode(self.qb, q_t)
        self.upload(qmm)

    def upload(self, qmm):
        buf = qmm.DeviceBuffer.from_numpy
        lay = (lambda a: a) if self.layout == "token" else (lambda a: a.swapaxes(1, 2))
        self.dk, self.dv = buf(lay(self.kb)), buf(lay(self.vb))
        self.dq, self.dt = buf(self.qb), buf(self.tables)
        self.dl, self.dr = buf(np.array(self.row_lens, np.int32)), buf(np.array(self.reqs, np.int32))
        self.cache = qmm.KVCache(self.dk, self.dv, self.c_t, self.n_pages, self.page, self.kv, self.dim, layout=self.layout,
                                 k_scale=self.k_scale, v_scale=self.v_scale)

    def run(self, qmm, out_t=F32, scale=None, attn=None, stream=None):
        attn = attn or qmm.PagedAttention(self.heads, self.kv, self.dim, self.q_t, out_t, scale=scale, window=self.window)
        R = len(self.reqs)
        print(f"attn rows={R} keys<={max(self.row_lens)} heads={self.heads}/{self.kv} dim={self.dim} q={self.q_t} cache={self.c_t} "
              f"page={self.page} {self.layout} window={self.window} out={out_t}", flush=True)
        do, dlse = qmm.DeviceBuffer(R * self.heads * self.dim * ref.SIZE[out_t]), qmm.DeviceBuffer(R * self.heads * 4)
        do.fill(0x7F, stream)
        dlse.fill(0x7F, stream)
        attn.run(self.cache, self.dq, do, self.dt, self.max_pages, self.dl, R, d_rows=self.dr if self.mapped else None,
                 requests=len(self.lens), d_lse=dlse, stream=stream)
        return (do.download(ref.BITS[out_t], (R, self.heads, self.dim), stream), dlse.download(np.float32, (R, self.heads), stream))

    def check(self, got, out_t=F32, scale=None, hidden=()):
        """hidden: (request, key) that no row sees."""
        scale = self.dim ** -0.5 if scale is None else scale
        out, lse = ref.decode(got[0], out_t), got[1].astype(np.float64)
        for j, (r, n) in enumerate(zip(self.reqs, self.row_lens)):
            n = max(0, min(n, len(self.keys[r]))) if 0 <= r < len(self.lens) else 0
            lo = max(0, n - self.window) if self.window else 0
            at = [i for i in range(lo, n) if (r, i) not in hidden]
            k, v = (self.keys[r][at], self.values[r][at]) if n else (np.zeros((0, self.kv, self.dim)),) * 2
            o, l, size, dots = ref.attention(self.q[j], k, v, scale)
            if not at:
                assert not out[j].any() and np.all(lse[j] == -np.inf), j
                continue
            o_tol, l_tol = ref.attention_bounds(o, size, dots, np.abs(v).max(), self.dim, self.q_t, out_t, len(at))
            l_tol = l_tol + 2.0 ** -22 * np.abs(l)
            assert np.all(np.abs(out[j] - o) <= o_tol), ("out", j, n, float(np.nanmax(np.abs(out[j] - o) / o_tol)), np.isnan(out[j]).sum())
            assert np.all(np.abs(lse[j] - l) <= l_tol), ("lse", j, n, float(np.max(np.abs(lse[j] - l) / l_tol)))


LENS = [1, 0, 7, 8, 9, 31, 32, 33, 64, 255, 256, 257, 300]


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("q_t,c_t", [(BF16, BF16), (F16, F16), (BF16, F8), (F16, F8)])
def test_types_and_dims(qmm, dim, q_t, c_t):
    for out_t in (F32, q_t):
        c = Case(qmm, LENS, 8, 2, dim, q_t, c_t, seed=dim + c_t)
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (3, 1), (7, 1), (16, 1), (17, 1), (32, 2), (40, 8), (96, 2), (64, 64)])
def test_head_layouts(qmm, heads, kv):
    c = Case(qmm, [5, 130, 0, 700], heads, kv, 64, seed=heads)
    c.check(c.run(qmm))
    c = Case(qmm, [77, 2000], heads, kv, 128, BF16, F8, seed=heads + 1)
    c.check(c.run(qmm))


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 256])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_pages_and_layouts(qmm, page, layout):
    c = Case(qmm, [1, 23, 24, 25, 500, 0, 1111], 6, 3, 64, page=page, layout=layout, seed=page, max_pages=1300 // page)
    c.check(c.run(qmm))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000])
def test_window(qmm, window):
    c = Case(qmm, [1, 0, 31, 32, 33, 64, 99, 100, 101, 500, 1500], 8, 2, 128, window=window, seed=window)
    c.check(c.run(qmm))
    c = Case(qmm, [9000], 8, 1, 64, F16, F16, window=window * 4, seed=window)
    c.check(c.run(qmm))


@pytest.mark.parametrize("lens", [[5000], [20001, 3, 0, 700], [257] * 3])
@pytest.mark.parametrize("heads,kv,dim,q_t,c_t", [(8, 1, 128, BF16, BF16), (32, 8, 128, F16, F16), (40, 2, 64, BF16, F8), (4, 4, 256, F16, F16),
                                                  (6, 2, 96, BF16, BF16), (5, 1, 192, BF16, F8)])
def test_rows_cut_into_parts(qmm, lens, heads, kv, dim, q_t, c_t):
    for out_t in (F32, q_t):
        c = Case(qmm, lens, heads, kv, dim, q_t, c_t, seed=len(lens) + dim)
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("R", [63, 64, 65, 130, 600])
def test_many_ragged_rows(qmm, R):
    rng = np.random.default_rng(R)
    lens = rng.integers(0, 60, R)
    lens[R // 2], lens[R - 1], lens[0] = 4000, 900, 0
    c = Case(qmm, [int(n) for n in lens], 8, 2, 64, seed=R)
    c.check(c.run(qmm))


def test_rows_of_requests(qmm):
    """Rows that share a request (a prompt's tokens), padding rows and requests outside."""
    lens = [40, 300, 2]
    reqs = [1] * 9 + [0] * 5 + [2, -1, 3, -2 ** 31, 2 ** 31 - 1]
    row_lens = list(range(290, 299)) + [1, 2, 38, 39, 40] + [2, 5, 5, 5, 5]
    c = Case(qmm, lens, 8, 2, 128, reqs=reqs, row_lens=row_lens, seed=8)
    c.check(c.run(qmm))


def test_lengths_outside(qmm):
    """Negative lengths are 0, lengths past the table are the table's."""
    c = Case(qmm, [48, 48, 48], 4, 2, 64, row_lens=[-1, -2 ** 31, 2 ** 31 - 1], reqs=[0, 1, 2], seed=9)
    c.check(c.run(qmm))


def test_pages_outside(qmm):
    """Keys on pages that the cache does not have are not seen, wherever they lie."""
    c = Case(qmm, [100, 64, 2100], 8, 2, 128, seed=10)
    hidden = set()
    for r, col, bad in ((0, 1, -1), (0, 6, 2 ** 31 - 1), (1, 0, c.n_pages), (1, 1, -5), (1, 2, -2 ** 31), (1, 3, -1), (2, 70, -1)):
        c.tables[r, col] = bad
        hidden |= {(r, i) for i in range(col * 16, col * 16 + 16)}
    c.upload(qmm)
    c.check(c.run(qmm), hidden=hidden)


@pytest.mark.parametrize("q_t", [BF16, F16])
def test_large_and_negative_scores(qmm, q_t):
    c = Case(qmm, [1, 50, 3000], 8, 2, 64, q_t, q_t, k_size=12.0, seed=13)
    for scale in (1.0, -0.5, 0.0):
        c.check(c.run(qmm, scale=scale), scale=scale)


def test_infinite_and_lowest_values(qmm):
    """Keys of the type's lowest value and of -inf get no weight; a row with nothing else is
    empty; +inf and NaN that are seen come out as NaN, in their heads alone."""
    lowest = 0xFF7F
    c = Case(qmm, [40, 40, 40, 40], 4, 2, 64, seed=14)
    c.q = np.abs(c.q) + 0.5
    c.qb = ref.encode(c.q, BF16)
    c.q = ref.decode(c.qb, BF16)

    def put(r, key, head, bits):
        c.kb[c.tables[r, key // 16], key % 16, head] = bits
    for key in range(0, 40, 3):
        for h in range(2):
            put(0, key, h, lowest)
            put(1, key, h, 0xFF80)
    for key in range(40):
        put(2, key, 0, 0xFF80)
    put(3, 17, 1, 0x7F80)
    c.upload(qmm)
    out, lse = c.run(qmm)
    out = ref.decode(out, F32)
    every_third = {(r, i) for r in (0, 1) for i in range(0, 40, 3)}
    good = Case.__new__(Case)
    good.__dict__.update(c.__dict__)
    good.reqs, good.row_lens = [0, 1], [40, 40]
    good.check((ref.encode(out[:2], F32), lse[:2]), hidden=every_third)
    assert not out[2, :2].any() and np.all(lse[2, :2] == -np.inf) and np.isfinite(out[2, 2:]).all() and np.isfinite(lse[2, 2:]).all()
    assert np.isfinite(out[3, :2]).all() and np.isnan(out[3, 2:]).all()


def test_interleaved_cache_and_strides(qmm):
    """Keys and values in one array [pages][tokens][2][heads][dim], strided q and out."""
    c = Case(qmm, [100, 7, 1400], 6, 2, 64, seed=15)
    both = np.stack([c.kb, c.vb], 2)
    d = qmm.DeviceBuffer.from_numpy(both)
    desc = c.cache.desc
    desc.d_k, desc.d_v = d.ptr, ctypes.c_void_p(d.ptr.value + 2 * 64 * 2)
    desc.page_stride, desc.token_stride, desc.head_stride = 16 * 2 * 2 * 64, 2 * 2 * 64, 64
    wide = np.full((3, 6 * 64 + 40), 0x7FC0, np.uint16)
    wide[:, :6 * 64] = c.qb.reshape(3, -1)
    dq, do = qmm.DeviceBuffer.from_numpy(wide), qmm.DeviceBuffer(3 * (6 * 64 + 8) * 4)
    do.fill(0x11)
    attn, dlse = qmm.PagedAttention(6, 2, 64), qmm.DeviceBuffer(3 * 6 * 4)
    print("attn interleaved, strided", flush=True)
    attn.run(c.cache, dq, do, c.dt, c.max_pages, c.dl, 3, d_lse=dlse, q_stride=wide.shape[1], out_stride=6 * 64 + 8)
    got = do.download(np.uint32, (3, 6 * 64 + 8))
    c.check((np.ascontiguousarray(got[:, :6 * 64]).reshape(3, 6, 64), dlse.download(np.float32, (3, 6))))
    assert np.all(got[:, 6 * 64:] == 0x11111111)
    attn.run(c.cache, dq, do, c.dt, c.max_pages, c.dl, 3, q_stride=wide.shape[1], out_stride=6 * 64 + 8)  # without lse
    assert np.array_equal(do.download(np.uint32, got.shape), got)


def test_offsets_past_32_bits(qmm):
    """Pages more than 4 GiB into the cache."""
    page, kv, dim = 256, 8, 128
    per_page = page * kv * dim * 2  # 512 KiB
    n_pages = (9 << 29) // per_page + 2  # 4.5 GiB
    c = Case(qmm, [600, 300], 16, kv, dim, page=page, seed=16)
    d = qmm.DeviceBuffer((n_pages + 64) * per_page)  # values from page 0 on, keys from page 64 on
    d_k = ctypes.c_void_p(d.ptr.value + 64 * per_page)
    shift = n_pages - c.n_pages
    print(f"attn over {n_pages * per_page} bytes", flush=True)
    for base, bits in ((d_k, c.kb), (d.ptr, c.vb)):
        src = qmm.DeviceBuffer.from_numpy(bits)
        qmm.stream_copy(type("At", (), dict(ptr=ctypes.c_void_p(base.value + shift * per_page), nbytes=src.nbytes)), src, src.nbytes)
    cache = qmm.KVCache(d, d, BF16, n_pages, page, kv, dim)
    cache.desc.d_k = d_k
    dt = qmm.DeviceBuffer.from_numpy((c.tables + np.int32(shift)) * (c.tables >= 0) * (c.tables < c.n_pages))
    attn = qmm.PagedAttention(16, kv, dim)
    do, dlse = qmm.DeviceBuffer(2 * 16 * dim * 4), qmm.DeviceBuffer(2 * 16 * 4)
    attn.run(cache, c.dq, do, dt, c.max_pages, c.dl, 2, d_lse=dlse)
    c.check((do.download(np.uint32, (2, 16, dim)), dlse.download(np.float32, (2, 16))))


def test_equal_calls_give_equal_bits(qmm):
    """Whatever workgroup ends last; on another stream; with a workspace that calls of other
    sizes used in between."""
    a = Case(qmm, [9000, 40, 3100], 16, 2, 128, seed=17)
    b = Case(qmm, [700, 8000], 8, 4, 64, F16, F16, seed=18)
    attn, other = qmm.PagedAttention(16, 2, 128), qmm.PagedAttention(8, 4, 64, F16, F32)
    big = attn.work if attn.work.nbytes >= other.work.nbytes else other.work
    attn.work = other.work = big
    first, second = a.run(qmm, attn=attn), b.run(qmm, attn=other)
    a.check(first)
    b.check(second)
    s = qmm.Stream()
    for i in range(6):
        st = s.handle if i % 2 else None
        for c, at, want in ((a, attn, first), (b, other, second)):
            got = c.run(qmm, attn=at, stream=st)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1].view(np.uint32), want[1].view(np.uint32)), i


def test_graph_replays(qmm):
    """A captured call, replayed with other lengths and queries in its buffers."""
    from openmini_qmm.hip_runtime import Graph
    c = Case(qmm, [4000, 50, 600], 8, 2, 128, seed=19)
    attn, s = qmm.PagedAttention(8, 2, 128), qmm.Stream()
    do, dlse = qmm.DeviceBuffer(3 * 8 * 128 * 4), qmm.DeviceBuffer(3 * 8 * 4)
    g = Graph(s.handle, lambda st: attn.run(c.cache, c.dq, do, c.dt, c.max_pages, c.dl, 3, d_lse=dlse, stream=st))
    for rep, lens in enumerate(([4000, 50, 600], [1, 0, 599], [3999, 33, 64], [0, 0, 0])):
        c.row_lens = lens
        c.dl.upload(np.array(lens, np.int32), s.handle)
        print(f"attn graph replay {rep}", flush=True)
        g.launch(s.handle)
        s.synchronize()
        got = do.download(np.uint32, (3, 8, 128)), dlse.download(np.float32, (3, 8))
        c.check(got)
        eager = c.run(qmm, attn=attn)
        assert np.array_equal(eager[0], got[0])


def test_no_rows(qmm):
    c = Case(qmm, [5], 4, 2, 64)
    attn = qmm.PagedAttention(4, 2, 64)
    attn.run(c.cache, c.dq, c.dq, c.dt, 1, c.dl, 0, requests=1)
    with pytest.raises(qmm.InvalidInput):
        attn.run(c.cache, c.dq, c.dq, c.dt, 1, c.dl, 1)  # out of fp32 in the place of q
    with pytest.raises(qmm.InvalidInput):
        attn.run(c.cache, c.dq, c.dq, c.dt, 1, c.dl, 1, d_rows=c.dr)
