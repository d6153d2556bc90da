"""Decode attention with tables as wide as the rows' keys and far wider: how rows are given to
waves depends on the most keys that a table can hold, the results do not, beyond rounding."""
import ctypes

import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8
from test_gpu_attn_decode import LENS, Case

pytestmark = pytest.mark.gpu
WIDE = 320  # columns of 16 keys: 5120 keys


@pytest.mark.parametrize("max_pages", [None, WIDE])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("q_t,c_t", [(BF16, BF16), (F16, F16), (BF16, F8), (F16, F8)])
def test_types_and_dims(qmm, dim, q_t, c_t, max_pages):
    for out_t in (F32, q_t):
        c = Case(qmm, LENS, 8, 2, dim, q_t, c_t, seed=dim + c_t + 1, max_pages=max_pages)
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("keys", [1, 31, 33, 255, 256, 257, 480, 511, 512, 513, 1023, 1024, 1025])
@pytest.mark.parametrize("R", [1, 7, 70])
def test_lengths_around_the_limits(qmm, R, keys):
    """Longest rows on both sides of the lengths at which the division changes."""
    rng = np.random.default_rng(R + keys)
    lens = rng.integers(0, keys + 1, R)
    lens[-1] = keys
    for kv, dim, c_t in ((1, 128, BF16), (3, 64, F8)):
        c = Case(qmm, [int(n) for n in lens], 6, kv, dim, BF16, c_t, seed=R + keys)
        c.check(c.run(qmm))


@pytest.mark.parametrize("heads,kv", [(1, 1), (17, 1), (40, 8), (96, 2), (128, 64)])
@pytest.mark.parametrize("R", [2, 3, 5, 9])
def test_rows_by_units(qmm, heads, kv, R):
    """Numbers of rows and units that do not divide a launch, up to 512 pairs and past them."""
    c = Case(qmm, [5, 130, 0, 200, 64, 31, 77, 256, 1][:R], heads, kv, 64, seed=heads + R)
    c.check(c.run(qmm))


@pytest.mark.parametrize("window", [1, 31, 32, 33, 100, 500])
@pytest.mark.parametrize("max_pages", [None, WIDE])
def test_windows(qmm, window, max_pages):
    c = Case(qmm, [1, 0, 31, 32, 33, 64, 99, 100, 101, 500, 1500], 8, 2, 128, window=window, seed=window, max_pages=max_pages)
    c.check(c.run(qmm))


def test_lengths_and_pages_outside_a_wide_table(qmm):
    c = Case(qmm, [100, 64, 300, 300], 8, 2, 128, seed=10, max_pages=WIDE, reqs=[0, 1, 2, 3, -1, 4], row_lens=[100, 64, 300, -7, 9, 9])
    hidden = set()
    for r, col, bad in ((0, 1, -1), (0, 6, 2 ** 31 - 1), (1, 0, c.n_pages), (1, 1, -5), (1, 2, -2 ** 31), (1, 3, -1), (2, 9, -1)):
        c.tables[r, col] = bad
        hidden |= {(r, i) for i in range(col * 16, col * 16 + 16)}
    c.upload(qmm)
    c.check(c.run(qmm), hidden=hidden)


def test_wide_and_narrow_agree(qmm):
    """To 2^-20 of the largest value: both are fp32 sums of the same products."""
    lens, outs = [300, 1, 17, 256], []
    for max_pages in (None, WIDE):
        c = Case(qmm, lens, 16, 4, 128, seed=5)
        if max_pages:
            wide = np.full((4, max_pages), -1, np.int32)
            wide[:, :c.max_pages] = c.tables
            c.tables, c.max_pages = wide, max_pages
            c.upload(qmm)
        outs.append(c.run(qmm))
        c.check(outs[-1])
    a, b = (ref.decode(o[0], F32) for o in outs)
    assert np.max(np.abs(a - b)) <= 2.0 ** -20 * np.max(np.abs(a))
    assert np.max(np.abs(outs[0][1] - outs[1][1])) <= 2.0 ** -20 * np.max(np.abs(outs[0][1]))


def test_offsets_past_32_bits_in_a_wide_table(qmm):
    """Pages more than 4 GiB into the cache, and a table of 16384 keys."""
    page, kv, dim = 256, 8, 128
    per_page = page * kv * dim * 2  # 512 KiB
    n_pages = (9 << 29) // per_page + 2  # 4.5 GiB
    c = Case(qmm, [600, 300], 16, kv, dim, page=page, seed=16, max_pages=64)
    shift = n_pages - c.n_pages
    d = qmm.DeviceBuffer((n_pages + 64) * per_page)  # values from page 0 on, keys from page 64 on
    d_k = ctypes.c_void_p(d.ptr.value + 64 * per_page)
    print(f"attn over {n_pages * per_page} bytes, wide table", flush=True)
    for base, bits in ((d_k, c.kb), (d.ptr, c.vb)):
        src = qmm.DeviceBuffer.from_numpy(bits)
        qmm.stream_copy(type("At", (), dict(ptr=ctypes.c_void_p(base.value + shift * per_page), nbytes=src.nbytes)), src, src.nbytes)
    cache = qmm.KVCache(d, d, BF16, n_pages, page, kv, dim)
    cache.desc.d_k = d_k
    inside = (c.tables >= 0) & (c.tables < c.n_pages)
    dt = qmm.DeviceBuffer.from_numpy(np.where(inside, c.tables, 0) + np.int32(shift))
    do, dlse = qmm.DeviceBuffer(2 * 16 * dim * 4), qmm.DeviceBuffer(2 * 16 * 4)
    qmm.PagedAttention(16, kv, dim).run(cache, c.dq, do, dt, c.max_pages, c.dl, 2, d_lse=dlse)
    c.check((do.download(np.uint32, (2, 16, dim)), dlse.download(np.float32, (2, 16))))


def test_graph_replays_of_short_rows(qmm):
    from openmini_qmm.hip_runtime import Graph
    c = Case(qmm, [300, 50, 170], 8, 2, 128, seed=19)
    attn, s = qmm.PagedAttention(8, 2, 128), qmm.Stream()
    do, dlse = qmm.DeviceBuffer(3 * 8 * 128 * 4), qmm.DeviceBuffer(3 * 8 * 4)
    g = Graph(s.handle, lambda st: attn.run(c.cache, c.dq, do, c.dt, c.max_pages, c.dl, 3, d_lse=dlse, stream=st))
    for rep, lens in enumerate(([300, 50, 170], [1, 0, 169], [299, 33, 64], [0, 0, 0])):
        c.row_lens = lens
        c.dl.upload(np.array(lens, np.int32), s.handle)
        print(f"attn graph replay {rep}", flush=True)
        g.launch(s.handle)
        s.synchronize()
        got = do.download(np.uint32, (3, 8, 128)), dlse.download(np.float32, (3, 8))
        c.check(got)
        assert np.array_equal(c.run(qmm, attn=attn)[0], got[0])


@pytest.mark.parametrize("R,kv,most", [(257, 1, 32), (130, 2, 31), (300, 2, 100), (513, 1, 128), (1030, 1, 60), (2100, 2, 64), (400, 4, 33)])
@pytest.mark.parametrize("dim,c_t", [(128, BF16), (64, F8), (256, BF16)])
def test_many_short_rows(qmm, R, kv, most, dim, c_t):
    """Rows of a few tiles, more than workgroups take whole: empty ones, whole ones, one key."""
    rng = np.random.default_rng(R + most)
    lens = rng.integers(0, most + 1, R)
    lens[rng.random(R) < 0.1] = 0
    lens[0], lens[R // 2], lens[R - 1] = 1, most, 0
    c = Case(qmm, [int(n) for n in lens], 4, kv, dim, BF16, c_t, seed=R)
    c.check(c.run(qmm))


def test_many_short_rows_of_requests_and_windows(qmm):
    """The same for rows that share requests, lie outside them, or see a window."""
    rng = np.random.default_rng(5)
    reqs = [int(r) for r in rng.integers(-1, 4, 700)]
    lens = [70, 3, 128, 40]
    row_lens = [int(rng.integers(-2, (lens[r] if r >= 0 else 128) + 1)) for r in reqs]
    c = Case(qmm, lens, 8, 1, 128, reqs=reqs, row_lens=row_lens, seed=6)
    c.check(c.run(qmm))
    c = Case(qmm, [int(n) for n in rng.integers(0, 900, 520)], 8, 1, 64, window=60, seed=7)
    c.check(c.run(qmm))
