"""Attention of single tokens over caches of 8-bit integers on the GPU, against 64 bits, at the
bounds of attn_ref.attention_bounds (the blocks' scales are two more roundings of 32 bits, of a
score and of a probability; the bounds have sixteen).  What no row sees is 127 under a scale
of NaN."""
import numpy as np
import pytest

import attn_ref as ref
import kv_i8_ref as kv
from attn_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu
I8 = kv.I8
LENS = [1, 0, 7, 8, 9, 31, 32, 33, 64, 255, 256, 257, 300]


class Case:
    def __init__(self, qmm, lens, heads, kv_heads, dim, q_t=BF16, reqs=None, row_lens=None, window=0, seed=0, **kw):
        self.c = kv.Paged(qmm, lens, kv_heads, dim, I8, seed=seed, **kw)
        self.heads, self.q_t, self.window = heads, q_t, window
        self.mapped = reqs is not None
        self.reqs = list(range(len(lens))) if reqs is None else list(reqs)
        self.row_lens = list(lens) if row_lens is None else list(row_lens)
        self.qb = ref.encode(self.c.rng.standard_normal((len(self.reqs), heads, dim)), q_t)
        self.q = ref.decode(self.qb, q_t)
        self.queries(qmm)

    def queries(self, qmm):
        buf = qmm.DeviceBuffer.from_numpy
        self.dq, self.dl, self.dr = buf(self.qb), buf(np.array(self.row_lens, np.int32)), buf(np.array(self.reqs, np.int32))

    def run(self, qmm, out_t=F32, scale=None, attn=None, stream=None):
        c, R = self.c, len(self.reqs)
        attn = attn or qmm.PagedAttention(self.heads, c.kv, c.dim, self.q_t, out_t, scale=scale, window=self.window)
        print(f"attn_i8 rows={R} keys<={max(self.row_lens)} heads={self.heads}/{c.kv} dim={c.dim} q={self.q_t} block={c.block} page={c.page} "
              f"{c.layout} window={self.window} out={out_t}", flush=True)
        do, dlse = qmm.DeviceBuffer(R * self.heads * c.dim * ref.SIZE[out_t]), qmm.DeviceBuffer(R * self.heads * 4)
        do.fill(0x7F, stream)
        dlse.fill(0x7F, stream)
        attn.run(c.cache, self.dq, do, c.d_tables, c.max_pages, self.dl, R, d_rows=self.dr if self.mapped else None,
                 requests=len(c.lens), d_lse=dlse, stream=stream)
        return do.download(ref.BITS[out_t], (R, self.heads, c.dim), stream), dlse.download(np.float32, (R, self.heads), stream)

    def check(self, got, out_t=F32, scale=None, hidden=(), skip=()):
        c = self.c
        scale = c.dim ** -0.5 if scale is None else scale
        out, lse = ref.decode(got[0], out_t), got[1].astype(np.float64)
        for j, (r, n) in enumerate(zip(self.reqs, self.row_lens)):
            if j in skip:
                continue
            n = max(0, min(n, c.max_pages * c.page)) if 0 <= r < len(c.lens) else 0
            at = [i for i in range(max(0, n - self.window) if self.window else 0, n) if (r, i) not in hidden]
            k, v = c.tokens(r, at) if at else (np.zeros((0, c.kv, c.dim)),) * 2
            o, l, size, dots = ref.attention(self.q[j], k, v, scale)
            if not at:
                assert not out[j].any() and np.all(lse[j] == -np.inf), j
                continue
            o_tol, l_tol = ref.attention_bounds(o, size, dots, np.abs(v).max(), c.dim, BF16, out_t, len(at))
            l_tol = l_tol + 2.0 ** -22 * np.abs(l)
            assert np.all(np.abs(out[j] - o) <= o_tol), ("out", j, n, float(np.nanmax(np.abs(out[j] - o) / o_tol)), np.isnan(out[j]).sum())
            assert np.all(np.abs(lse[j] - l) <= l_tol), ("lse", j, n, float(np.max(np.abs(lse[j] - l) / l_tol)))


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("q_t", [BF16, F16])
@pytest.mark.parametrize("block,page", [(8, 8), (16, 16), (32, 32)])
def test_types_and_dims(qmm, dim, q_t, block, page):
    for out_t in (F32, q_t):
        c = Case(qmm, LENS, 8, 2, dim, q_t, block=block, page=page, seed=dim + block)
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (7, 1), (16, 1), (17, 1), (40, 8), (96, 2)])
def test_head_layouts(qmm, heads, kv_heads):
    for dim, lens in ((64, [5, 130, 0, 700]), (128, [77, 2000])):
        c = Case(qmm, lens, heads, kv_heads, dim, seed=heads)
        c.check(c.run(qmm))


@pytest.mark.parametrize("block,page", [(8, 24), (8, 40), (16, 64), (32, 160), (32, 256)])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_pages_and_layouts(qmm, block, page, layout):
    c = Case(qmm, [1, 23, 24, 25, 500, 0, 1111], 6, 3, 64, block=block, page=page, layout=layout, seed=page, max_pages=1300 // page + 1)
    c.check(c.run(qmm))


@pytest.mark.parametrize("window", [1, 2, 31, 33, 100, 1000])
def test_window(qmm, window):
    c = Case(qmm, [1, 0, 31, 32, 33, 64, 99, 100, 101, 500, 1500], 8, 2, 128, window=window, seed=window)
    c.check(c.run(qmm))
    c = Case(qmm, [9000], 8, 1, 64, F16, window=window * 4, seed=window)
    c.check(c.run(qmm))


@pytest.mark.parametrize("lens", [[5000], [20001, 3, 0, 700], [257] * 3])
@pytest.mark.parametrize("heads,kv_heads,dim,q_t", [(8, 1, 128, BF16), (32, 8, 128, F16), (40, 2, 64, BF16), (4, 4, 256, F16), (6, 2, 96, BF16),
                                                    (5, 1, 192, BF16)])
def test_rows_cut_into_parts(qmm, lens, heads, kv_heads, dim, q_t):
    for out_t in (F32, q_t):
        c = Case(qmm, lens, heads, kv_heads, dim, q_t, block=8 if dim == 64 else 16, seed=len(lens) + dim)
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("R", [65, 600])
def test_many_ragged_rows(qmm, R):
    lens = np.random.default_rng(R).integers(0, 60, R)
    lens[R // 2], lens[R - 1], lens[0] = 4000, 900, 0
    c = Case(qmm, [int(n) for n in lens], 8, 2, 64, seed=R)
    c.check(c.run(qmm))


def test_rows_of_requests_and_lengths_outside(qmm):
    c = Case(qmm, [40, 300, 2], 8, 2, 128, reqs=[1] * 9 + [0] * 3 + [2, -1, 3, 2 ** 31 - 1], row_lens=list(range(290, 299)) + [1, 39, 40] + [2, 5, 5, 5],
             seed=8)
    c.check(c.run(qmm))
    c = Case(qmm, [48, 48, 48], 4, 2, 64, row_lens=[-1, -2 ** 31, 2 ** 31 - 1], reqs=[0, 1, 2], seed=9)
    c.check(c.run(qmm))


def test_pages_outside(qmm):
    c = Case(qmm, [100, 64, 2100], 8, 2, 128, seed=10)
    hidden = set()
    for r, col, bad in ((0, 1, -1), (0, 6, 2 ** 31 - 1), (1, 0, c.c.n_pages), (1, 1, -5), (1, 2, -2 ** 31), (1, 3, -1), (2, 70, -1)):
        c.c.tables[r, col] = bad
        hidden |= {(r, i) for i in range(col * 16, col * 16 + 16)}
    c.c.upload(qmm)
    c.check(c.run(qmm), hidden=hidden)


def test_scales_of_all_sizes(qmm):
    """Zero (a block of zeros), the least that is written, and 2^30 times the others; large and
    negative scores."""
    c = Case(qmm, [300, 200], 8, 2, 64, seed=11)
    p = c.c
    for i in range(2):
        p.scales[i][p.tables[0, 2], 0, 0] = 0
        p.scales[i][p.tables[0, 3], 0, 1] = 2.0 ** -40
        p.scales[i][p.tables[1, 4], 0] = 0
    p.scales[1][p.tables[0, 7], 0, 0] *= 2.0 ** 30
    p.upload(qmm)
    for scale in (None, 3.0, -0.5, 0.0):
        c.check(c.run(qmm, scale=scale), scale=scale)


def test_scales_without_a_number(qmm):
    """A NaN scale of keys makes the heads that see the block NaN, one of values their outputs alone;
    rows that end before it, or whose window begins behind it, are as ever."""
    lens = [100] * 5
    for window in (0, 40):
        c = Case(qmm, lens, 4, 2, 64, row_lens=[32, 100, 100, 100, 100], reqs=[0, 0, 1, 2, 3], window=window, seed=12)
        p = c.c
        p.scales[0][p.tables[0, 2], 0, 0] = np.nan      # keys 32 - 47 of request 0
        p.scales[1][p.tables[1, 5], 0, 1] = np.nan      # values 80 - 95 of request 1
        p.scales[0][p.tables[2, 0], 0] = np.inf         # keys 0 - 15 of request 2: 0 times inf
        p.bits[0][p.tables[2, 0]] = 0
        p.scales[1][p.tables[3, 6], 0, 0] = np.inf
        p.upload(qmm)
        got = c.run(qmm)
        out = ref.decode(got[0], F32)
        c.check(got, skip=(1, 2, 3, 4) if not window else (2, 4))
        if not window:
            assert np.isnan(out[1, :2]).all() and np.isnan(got[1][1, :2]).all() and np.isfinite(out[1, 2:]).all()
            assert np.isnan(out[3]).all()
        assert np.isnan(out[2, 2:]).all() and np.isfinite(got[1][2]).all() and np.isfinite(out[2, :2]).all()
        assert not np.isfinite(out[4, :2]).any() and np.isfinite(out[4, 2:]).all()


def test_sinks(qmm):
    """A first key far above the others whose value is nearly zero: the output is made of
    probabilities far below it."""
    for q_t in (BF16, F16):
        c = Case(qmm, [3000], 4, 1, 64, q_t, seed=13)
        p = c.c
        c.q = np.abs(c.q) + 0.5
        c.qb = ref.encode(c.q, q_t)
        c.q = ref.decode(c.qb, q_t)
        c.queries(qmm)
        page = int(p.tables[0, 0])
        p.bits[0][page, 0], p.bits[1][page, 0] = 127, 0
        for nats in (12.0, 20.0, 35.0):
            # the first block's scale, so that the first key's score is about `nats`
            p.scales[0][page, 0] = nats / (np.abs(c.q[0, 0]).sum() * 127 * 64 ** -0.5)
            p.upload(qmm)
            c.check(c.run(qmm))


def test_strided_scales_and_interleaved_caches(qmm):
    """Keys and values in one array, and their scales in one."""
    import ctypes
    c = Case(qmm, [100, 7, 1400], 6, 2, 64, page=32, block=8, seed=15)
    p = c.c
    d = qmm.DeviceBuffer.from_numpy(np.stack(p.bits, 2))                 # [pages][32][2][2][64]
    ds = qmm.DeviceBuffer.from_numpy(np.stack(p.scales, 1).swapaxes(2, 3).copy())  # [pages][2][heads][blocks]
    desc, sc = p.cache.desc, p.cache.scales
    desc.d_k, desc.d_v = d.ptr, ctypes.c_void_p(d.ptr.value + 2 * 64)
    desc.page_stride, desc.token_stride, desc.head_stride = 32 * 256, 256, 64
    sc.d_k, sc.d_v = ds.ptr, ctypes.c_void_p(ds.ptr.value + 2 * 4 * 4)
    sc.page_stride, sc.block_stride, sc.head_stride = 16, 1, 4
    c.check(c.run(qmm))


def test_offsets_past_32_bits(qmm):
    page, kv_heads, dim = 256, 8, 128
    per_page, per_scales = page * kv_heads * dim, 8 * kv_heads * 4
    n_pages = (9 << 29) // per_page + 2
    c = Case(qmm, [600, 300], 16, kv_heads, dim, page=page, block=32, seed=16)
    p = c.c
    d, ds = [qmm.DeviceBuffer(n_pages * per_page) for _ in range(2)], [qmm.DeviceBuffer(n_pages * per_scales) for _ in range(2)]
    shift = n_pages - p.n_pages
    for i in range(2):
        for buf, src, each in ((d[i], p.bits[i], per_page), (ds[i], p.scales[i], per_scales)):
            qmm.stream_copy(kv.at_page(buf, shift * each, src.nbytes), qmm.DeviceBuffer.from_numpy(src), src.nbytes)
    p.cache = qmm.KVCache(d[0], d[1], I8, n_pages, page, kv_heads, dim, block=32, d_k_scales=ds[0], d_v_scales=ds[1])
    p.d_tables = qmm.DeviceBuffer.from_numpy(np.where((p.tables >= 0) & (p.tables < p.n_pages), p.tables + shift, -1).astype(np.int32))
    c.check(c.run(qmm))


def test_large_caches_and_equal_bits(qmm):
    """Read past the caches (160 MB under tables of 20000 columns): the same bits as from a small one;
    equal calls give equal bits, on other streams and after calls of other sizes."""
    small = Case(qmm, [3000, 50, 600], 8, 2, 128, seed=19, max_pages=20000)
    large = Case(qmm, [3000, 50, 600], 8, 2, 128, seed=19, max_pages=20000, extra=3)
    p = large.c
    per_page, n = 16 * 2 * 128, 20000
    d, ds = [qmm.DeviceBuffer(n * per_page) for _ in range(2)], [qmm.DeviceBuffer(n * 8) for _ in range(2)]
    for i in range(2):
        d[i].fill(0x7F)
        ds[i].fill(0xFF)
        for buf, src in ((d[i], p.bits[i]), (ds[i], p.scales[i])):
            buf.upload(src)
    p.cache = qmm.KVCache(d[0], d[1], I8, n, 16, 2, 128, block=16, d_k_scales=ds[0], d_v_scales=ds[1])
    p.d_tables = qmm.DeviceBuffer.from_numpy(np.where((p.tables >= 0) & (p.tables < p.n_pages), p.tables, -1).astype(np.int32))
    first = small.run(qmm)
    small.check(first)
    attn, other, st = qmm.PagedAttention(8, 2, 128), Case(qmm, [700, 8000], 8, 2, 128, F16, seed=3), qmm.Stream()
    second = qmm.PagedAttention(8, 2, 128, F16, F32)
    second.work = attn.work
    for i in range(4):
        got = large.run(qmm, attn=attn, stream=st.handle if i % 2 else None)
        assert np.array_equal(got[0], first[0]) and np.array_equal(got[1], first[1])
        other.check(other.run(qmm, attn=second))


def test_graph_replays(qmm):
    from openmini_qmm.hip_runtime import Graph
    c = Case(qmm, [4000, 50, 600], 8, 2, 128, seed=19)
    attn, s = qmm.PagedAttention(8, 2, 128), qmm.Stream()
    do, dlse = qmm.DeviceBuffer(3 * 8 * 128 * 4), qmm.DeviceBuffer(3 * 8 * 4)
    g = Graph(s.handle, lambda st: attn.run(c.c.cache, c.dq, do, c.c.d_tables, c.c.max_pages, c.dl, 3, d_lse=dlse, stream=st))
    for rep, lens in enumerate(([4000, 50, 600], [1, 0, 599], [3999, 33, 64], [0, 0, 0])):
        c.row_lens = lens
        c.dl.upload(np.array(lens, np.int32), s.handle)
        print(f"attn_i8 graph replay {rep}", flush=True)
        g.launch(s.handle)
        s.synchronize()
        got = do.download(np.uint32, (3, 8, 128)), dlse.download(np.float32, (3, 8))
        c.check(got)
        assert np.array_equal(c.run(qmm, attn=attn)[0], got[0])
