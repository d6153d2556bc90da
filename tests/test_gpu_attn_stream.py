"""Decode attention over caches and tables so large that keys and values are read past the
caches: the same inputs as elsewhere, in pages spread over a cache of 160 MB, under tables
of 20000 columns."""
import ctypes

import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8
from test_gpu_attn_decode import LENS, Case

pytestmark = pytest.mark.gpu
COLUMNS = 20000


class Large(Case):
    """A Case whose pages lie anywhere in a cache of `mega` MB a side, full of the type's NaN."""

    def upload(self, qmm, mega=80, shift=0):
        per_page = self.page * self.kv * self.dim * ref.SIZE[self.c_t]
        n = max(mega * 1000000 // per_page, self.n_pages)
        to = np.random.default_rng(1).permutation(n)[:self.n_pages].astype(np.int32)
        buf = qmm.DeviceBuffer.from_numpy
        self.dk, self.dv = qmm.DeviceBuffer(n * per_page + shift), qmm.DeviceBuffer(n * per_page + shift)
        lay = (lambda a: a) if self.layout == "token" else (lambda a: a.swapaxes(1, 2))
        for d, bits in ((self.dk, self.kb), (self.dv, self.vb)):
            d.fill(0xFF)  # NaN in every type
            for page in range(self.n_pages):
                at = type("At", (), dict(ptr=ctypes.c_void_p(d.ptr.value + shift + int(to[page]) * per_page), nbytes=per_page))
                qmm.stream_copy(at, buf(np.ascontiguousarray(lay(bits[page:page + 1]))), per_page)
        inside = (self.tables >= 0) & (self.tables < self.n_pages)
        self.dq, self.dt = buf(self.qb), buf(np.where(inside, to[np.where(inside, self.tables, 0)], self.tables.clip(None, -1)).astype(np.int32))
        self.dl, self.dr = buf(np.array(self.row_lens, np.int32)), buf(np.array(self.reqs, np.int32))
        self.cache = qmm.KVCache(self.dk, self.dv, self.c_t, n, self.page, self.kv, self.dim, layout=self.layout,
                                 k_scale=self.k_scale, v_scale=self.v_scale)
        self.cache.desc.d_k = ctypes.c_void_p(self.dk.ptr.value + shift)
        self.cache.desc.d_v = ctypes.c_void_p(self.dv.ptr.value + shift)


@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("q_t,c_t", [(BF16, BF16), (F16, F16), (BF16, F8), (F16, F8)])
def test_types_and_dims(qmm, dim, q_t, c_t, layout):
    c = Large(qmm, LENS, 8, 2, dim, q_t, c_t, seed=dim + c_t, max_pages=COLUMNS, layout=layout)
    c.check(c.run(qmm))


@pytest.mark.parametrize("shift", [0, 16, 64])
def test_alignment(qmm, shift):
    """Caches that begin inside a line."""
    c = Large(qmm, [900, 33, 0, 2000], 8, 2, 128, seed=2, max_pages=COLUMNS)
    c.upload(qmm, shift=shift)
    c.check(c.run(qmm))


def test_long_rows_windows_and_heads(qmm):
    for heads, kv, lens, window in ((16, 1, [30001], 0), (32, 1, [9000, 5], 0), (8, 2, [20000, 300, 0], 4100), (4, 4, [7000] * 2, 0)):
        c = Large(qmm, lens, heads, kv, 128, BF16, F8, seed=heads, max_pages=COLUMNS, window=window)
        c.check(c.run(qmm))


def test_rows_that_share_a_request(qmm):
    c = Large(qmm, [60, 300], 8, 2, 128, reqs=[1] * 6 + [0], row_lens=[295, 296, 297, 298, 299, 300, 60], seed=4, max_pages=COLUMNS)
    c.check(c.run(qmm))


def test_pages_outside(qmm):
    c = Large(qmm, [100, 64, 2100], 8, 2, 128, seed=10, max_pages=COLUMNS)
    hidden = set()
    for r, col, bad in ((0, 1, -1), (0, 6, -2 ** 31), (1, 0, -7), (1, 1, -5), (1, 2, -2 ** 31), (1, 3, -1), (2, 70, -1)):
        c.tables[r, col] = bad
        hidden |= {(r, i) for i in range(col * 16, col * 16 + 16)}
    c.upload(qmm)
    c.check(c.run(qmm), hidden=hidden)


def test_equal_to_a_small_cache_and_replays(qmm):
    """How loads are marked changes no bit: a cache too small for it, the same columns."""
    from openmini_qmm.hip_runtime import Graph
    a = Case(qmm, [3000, 50, 600], 8, 2, 128, seed=19, max_pages=COLUMNS)
    b = Large(qmm, [3000, 50, 600], 8, 2, 128, seed=19, max_pages=COLUMNS)
    first, second = a.run(qmm), b.run(qmm)
    b.check(second)
    assert np.array_equal(first[0], second[0]) and np.array_equal(first[1], second[1])
    attn, s = qmm.PagedAttention(8, 2, 128), qmm.Stream()
    do = qmm.DeviceBuffer(3 * 8 * 128 * 4)
    g = Graph(s.handle, lambda st: attn.run(b.cache, b.dq, do, b.dt, b.max_pages, b.dl, 3, stream=st))
    for rep in range(3):
        print(f"attn graph replay {rep}", flush=True)
        g.launch(s.handle)
        s.synchronize()
        assert np.array_equal(do.download(np.uint32, (3, 8, 128)), second[0])
        assert np.array_equal(b.run(qmm, attn=attn)[0], second[0])
