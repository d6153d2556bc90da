"""Reading a paged cache back on the GPU: elements are exact products of an element and its scale
in 32 bits, rounded once to the output's type, so results are compared bit for bit."""
import numpy as np
import pytest

import attn_ref as ref
import kv_i8_ref as kv
from attn_ref import BF16, F16, F32, F8

pytestmark = pytest.mark.gpu
I8 = kv.I8


def _want(c, r, at, i, out_t):
    """Elements of tokens `at` of request r in out_t's bits: fp32 products first."""
    rows = np.zeros((len(at), c.kv, c.dim), np.float32)
    for j, p in enumerate(at):
        if not 0 <= p < c.max_pages * c.page:
            continue
        page = c.tables[r, p // c.page]
        if not 0 <= page < c.n_pages:
            continue
        b = c.bits[i][page, p % c.page]
        if c.c_t == I8:
            rows[j] = b.astype(np.float32) * c.scales[i][page, p % c.page // c.block][:, None]
        else:
            rows[j] = ref.decode(b, c.c_t).astype(np.float32) * np.float32((c.k_scale, c.v_scale)[i])
    return rows.view(np.uint32) if out_t == F32 else ref.encode(rows, out_t)


def _run(qmm, c, spans, out_t, pad=0, k=True, v=True, stream=None, first=True):
    """spans: (first, count) of each request; rows behind them are not the call's."""
    starts = np.concatenate([[0], np.cumsum([n for _, n in spans])]).astype(np.int32)
    total = int(starts[-1])
    row = c.kv * c.dim + pad
    print(f"read tokens={total} kv={c.kv} dim={c.dim} cache={c.c_t} page={c.page} block={c.block} {c.layout} out={out_t}", flush=True)
    outs = [qmm.DeviceBuffer((total + 5) * row * ref.SIZE[out_t]) for _ in range(2)]
    for o in outs:
        o.fill(0x5A, stream)
    buf = qmm.DeviceBuffer.from_numpy
    c.cache.read(c.d_tables, c.max_pages, buf(starts), len(spans), total + 5, outs[0] if k else None, outs[1] if v else None, out_t,
                 d_first=buf(np.array([f for f, _ in spans], np.int32)) if first else None, k_stride=row, v_stride=row, stream=stream)
    got = [o.download(ref.BITS[out_t], (total + 5, row), stream) for o in outs]
    untouched = np.frombuffer(b"\x5a" * ref.SIZE[out_t], ref.BITS[out_t])[0]
    for i, on in enumerate((k, v)):
        if not on:
            assert np.all(got[i] == untouched)
            continue
        assert np.all(got[i][total:] == untouched) and np.all(got[i][:, c.kv * c.dim:] == untouched)
        for r, (f, n) in enumerate(spans):
            a = got[i][starts[r]:starts[r + 1], :c.kv * c.dim].reshape(n, c.kv, c.dim)
            b = _want(c, r, range(f, f + n), i, out_t)
            nan = np.isnan(ref.decode(b, out_t))
            assert np.array_equal(np.isnan(ref.decode(a, out_t)), nan) and np.array_equal(a[~nan], b[~nan]), (i, r)
    return got


@pytest.mark.parametrize("c_t", [I8, F8, F16, BF16])
@pytest.mark.parametrize("out_t", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_types_and_layouts(qmm, c_t, out_t, layout):
    c = kv.Paged(qmm, [40, 1, 0, 130, 16], 3, 64, c_t, page=16, block=8, layout=layout, seed=c_t)
    _run(qmm, c, [(0, 40), (0, 1), (0, 0), (7, 100), (15, 1)], out_t)


@pytest.mark.parametrize("kv_heads,dim,page,block", [(1, 16, 8, 8), (8, 128, 64, 32), (2, 256, 24, 8), (5, 96, 160, 32), (1, 192, 16, 16),
                                                     (32, 64, 256, 16), (1, 512, 32, 32), (2, 48, 32, 16)])
def test_sizes(qmm, kv_heads, dim, page, block):
    c = kv.Paged(qmm, [page * 2 + 3, 17], kv_heads, dim, I8, page, block, seed=dim)
    _run(qmm, c, [(1, page * 2), (0, 17)], BF16, pad=8)
    _run(qmm, c, [(1, page * 2), (0, 17)], F32, v=False)
    _run(qmm, c, [(0, 30), (0, 9)], F16, k=False, first=False)


def test_odd_dims(qmm):
    """Heads of 8 and 24, whose rows are whole 16 bytes in 16-bit caches."""
    for dim in (8, 24):
        c = kv.Paged(qmm, [19, 17], 2, dim, BF16, 8, seed=dim)
        _run(qmm, c, [(1, 16), (0, 17)], F32)
        _run(qmm, c, [(1, 16), (0, 17)], BF16, pad=8)


def test_places_outside(qmm):
    """Before the first token, past the table, on pages that the cache does not have: zeros."""
    c = kv.Paged(qmm, [64, 64, 64], 2, 64, I8, seed=3)
    c.tables[0, 1], c.tables[1, 0], c.tables[1, 3] = -1, c.n_pages, -2 ** 31
    c.upload(qmm)
    got = _run(qmm, c, [(-9, 80), (0, 70), (2 ** 31 - 3, 5)], F32)
    assert not got[0][:9].any() and not got[1][150:155].any()


def test_many_requests(qmm):
    """More requests than a wave has lanes, most of them empty."""
    rng = np.random.default_rng(4)
    lens = [int(n) for n in rng.integers(0, 30, 500)]
    c = kv.Paged(qmm, lens, 1, 32, I8, page=8, block=8, seed=5)
    spans = [(0, 0) if n == 0 or rng.random() < 0.6 else (int(rng.integers(0, n)), 1) for n in lens]
    _run(qmm, c, spans, F16)


def test_odd_starts(qmm):
    """Rows before the first run and between runs stay as they were; starts that do not rise, or lie
    outside, reach no row that is not there."""
    c = kv.Paged(qmm, [20, 20], 1, 64, I8, seed=6)
    buf = qmm.DeviceBuffer.from_numpy
    for starts in ([3, 5, 9], [0, 0, 0], [-5, 2, 2 ** 31 - 1], [9, 4, 1], [2 ** 31 - 1, -1, -2 ** 31]):
        o = qmm.DeviceBuffer(10 * 64 * 4)
        o.fill(0x5A)
        print(f"read starts={starts}", flush=True)
        c.cache.read(c.d_tables, c.max_pages, buf(np.array(starts, np.int32)), 2, 10, o, None, F32)
        got = o.download(np.uint32, (10, 64))
        if starts[0] == 3:
            assert np.all(got[:3] == 0x5A5A5A5A) and np.all(got[9:] == 0x5A5A5A5A)
            assert np.array_equal(got[3:5], _want(c, 0, range(2), 0, F32)[:, 0]) and np.array_equal(got[5:9], _want(c, 1, range(4), 0, F32)[:, 0])
        if starts == [0, 0, 0]:
            assert np.all(got == 0x5A5A5A5A)


def test_scales_without_a_number(qmm):
    c = kv.Paged(qmm, [40], 2, 64, I8, seed=7)
    p = int(c.tables[0, 1])
    c.scales[0][p, 0, 1], c.scales[1][p, 0, 0] = np.nan, np.inf
    c.bits[1][p, 3, 0] = 0
    c.upload(qmm)
    got = _run(qmm, c, [(0, 40)], F32)
    k = got[0].view(np.float32).reshape(-1, 2, 64)[:40]
    assert np.isnan(k[16:32, 1]).all() and np.isfinite(k[:, 0]).all() and np.isfinite(k[:16]).all()


def test_streams_and_replays(qmm):
    from openmini_qmm.hip_runtime import Graph
    c = kv.Paged(qmm, [100, 33], 4, 128, I8, seed=8)
    st = qmm.Stream()
    first = _run(qmm, c, [(0, 100), (0, 33)], BF16, stream=st.handle)
    starts = qmm.DeviceBuffer.from_numpy(np.array([0, 100, 133], np.int32))
    outs = [qmm.DeviceBuffer(133 * 512 * 2) for _ in range(2)]
    g = Graph(st.handle, lambda h: c.cache.read(c.d_tables, c.max_pages, starts, 2, 133, outs[0], outs[1], BF16, stream=h))
    for _ in range(3):
        for o in outs:
            o.fill(0, st.handle)
        g.launch(st.handle)
        st.synchronize()
        for o, f in zip(outs, first):
            assert np.array_equal(o.download(np.uint16, (133, 512)), f[:133])


def test_offsets_past_32_bits(qmm):
    """Pages more than 4 GiB into the cache, outputs past 4 GiB."""
    page, kv_heads, dim = 256, 8, 128
    per_page = page * kv_heads * dim
    n_pages = (9 << 29) // per_page + 1
    c = kv.Paged(qmm, [600], kv_heads, dim, I8, page=page, block=32, seed=9)
    d, ds = qmm.DeviceBuffer(n_pages * per_page), qmm.DeviceBuffer(n_pages * 8 * kv_heads * 4)
    shift = n_pages - c.n_pages
    for buf, src, each in ((d, c.bits[0], per_page), (ds, c.scales[0], 8 * kv_heads * 4)):
        qmm.stream_copy(kv.at_page(buf, shift * each, src.nbytes), qmm.DeviceBuffer.from_numpy(src), src.nbytes)
    whole = qmm.KVCache(d, d, I8, n_pages, page, kv_heads, dim, block=32, d_k_scales=ds, d_v_scales=ds)
    tables = np.where((c.tables >= 0) & (c.tables < c.n_pages), c.tables + shift, -1).astype(np.int32)
    stride = 2 << 20  # elements a row: 600 rows of 8 MiB
    o = qmm.DeviceBuffer(599 * stride * 4 + kv_heads * dim * 4)
    print("read into 4.7 GiB", flush=True)
    whole.read(qmm.DeviceBuffer.from_numpy(tables), c.max_pages, qmm.DeviceBuffer.from_numpy(np.array([0, 600], np.int32)), 1, 600, o, None,
               F32, k_stride=stride)
    for j in (0, 255, 256, 599):
        back = qmm.DeviceBuffer(kv_heads * dim * 4)
        qmm.stream_copy(back, kv.at_page(o, j * stride * 4, back.nbytes), back.nbytes)
        assert np.array_equal(back.download(np.uint32, (1, kv_heads, dim)), _want(c, 0, [j], 0, F32)), j


def test_refusals(qmm):
    c = kv.Paged(qmm, [5], 1, 64, I8)
    d = qmm.DeviceBuffer(1 << 12)
    with pytest.raises(qmm.QmmError, match="both null"):
        c.cache.read(c.d_tables, c.max_pages, d, 1, 1, None, None, F32)
    with pytest.raises(qmm.QmmError, match="requests"):
        c.cache.read(c.d_tables, c.max_pages, d, 0, 0, d, d, F32)
    c.cache.read(c.d_tables, c.max_pages, d, 1, 0, d, d, F32)  # no tokens
