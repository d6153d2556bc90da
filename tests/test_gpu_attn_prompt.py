"""Attention of runs of query tokens on the GPU, against 64 bits.  What no row sees holds NaN."""
import numpy as np
import pytest

import attn_ref as ref
import kv_i8_ref as kv
from attn_ref import BF16, F16, F32, F8

pytestmark = pytest.mark.gpu
I8 = kv.I8
TYPES = [(BF16, I8), (F16, I8), (BF16, BF16), (F16, F16), (BF16, F8), (F16, F8)]


def bounds(o, size, dots, v_most, dim, q_t, c_t, out_t, n):
    """How far the kernel may be off, worst case.  A score: dim products added in 32 bits, scaled,
    the logarithm of a scale of up to 2^60 added (60 2^-24 and the sum's rounding), the maximum's
    difference and the exponential: dim + 16 roundings of 2^-24 of the sum of magnitudes, and 2^-17;
    an error e of the scores moves the output by at most 2 e sum p |v|.  A probability is rounded
    once, by 2^-8 of it in bf16 (bf16 caches) or 2^-11 in fp16: 2^11 at a row's base, at most 2^4 above
    which its largest lies, so that half of the least unit, 2^-25, is 2^-36 of the largest; as parts, for fp32 outputs, 2^-21 stays.  Sums in 32 bits of n terms,
    32 at a time, of the steps and of the splits."""
    e = (dim + 16) * 2.0 ** -24 * dots + (2.0 ** -17 if c_t == I8 else 2.0 ** -22)
    part = 2.0 ** -21 if out_t == F32 else 2.0 ** -8 if c_t == BF16 else 2.0 ** -11
    d = (2 * e[:, None] + part + (n / 32 + 64) * 2.0 ** -24) * size + n * 2.0 ** -36 * v_most
    d = d + ref.ROUND[out_t] * (np.abs(o) + d) + ref.TINY[out_t]
    return d, e + (n / 32 + 64) * 2.0 ** -24 + 2.0 ** -22


class Case:
    """Requests that hold `held` tokens and have runs of `new` query tokens; each sees the keys up to
    its own unless `lens` says otherwise.  gaps: rows of no request before each run."""

    def __init__(self, qmm, held, new, heads, kv_heads, dim, q_t=BF16, c_t=I8, window=0, seed=0, lens=None, gaps=None, q_size=1.0, **kw):
        self.c = c = kv.Paged(qmm, [h + n for h, n in zip(held, new)], kv_heads, dim, c_t, seed=seed, **kw)
        self.heads, self.q_t, self.window = heads, q_t, window
        self.starts, self.runs, at = [], [], 0
        for r, n in enumerate(new):
            at += gaps[r] if gaps else 0
            self.runs.append((at, n))
            at += n
        # runs follow each other: a gap belongs to a request of its own that has no keys (lens 0)
        assert not gaps
        self.starts = [s for s, _ in self.runs] + [at]
        self.rows = at + 3
        self.lens = [h + i + 1 for h, n in zip(held, new) for i in range(n)] + [5] * 3 if lens is None else list(lens) + [5] * 3
        self.qb = ref.encode(c.rng.standard_normal((self.rows, heads, dim)) * q_size, q_t)
        self.q = ref.decode(self.qb, q_t)
        self.queries(qmm)

    def queries(self, qmm):
        buf = qmm.DeviceBuffer.from_numpy
        self.dq, self.dl, self.ds = buf(self.qb), buf(np.array(self.lens, np.int32)), buf(np.array(self.starts, np.int32))

    def run(self, qmm, out_t=None, scale=None, attn=None, stream=None, requests=None):
        c = self.c
        out_t = self.q_t if out_t is None else out_t
        attn = attn or qmm.PromptAttention(self.heads, c.kv, c.dim, self.q_t, out_t, scale=scale, window=self.window)
        print(f"prompt rows={self.rows} runs={len(self.runs)} keys<={max(self.lens)} heads={self.heads}/{c.kv} dim={c.dim} q={self.q_t} "
              f"cache={c.c_t} block={c.block} page={c.page} {c.layout} window={self.window} out={out_t}", flush=True)
        do, dlse = qmm.DeviceBuffer(self.rows * self.heads * c.dim * ref.SIZE[out_t]), qmm.DeviceBuffer(self.rows * self.heads * 4)
        do.fill(0x5A, stream)
        dlse.fill(0x5A, stream)
        attn.run(c.cache, self.dq, do, c.d_tables, c.max_pages, self.ds, self.dl, self.rows, len(self.runs) if requests is None else requests,
                 d_lse=dlse, stream=stream)
        return (do.download(ref.BITS[out_t], (self.rows, self.heads, c.dim), stream),
                dlse.download(np.float32, (self.rows, self.heads), stream))

    def check(self, got, out_t=None, scale=None, hidden=(), skip=(), rows=None):
        """rows: those that are compared (all); those of no run must be as they were."""
        c = self.c
        out_t = self.q_t if out_t is None else out_t
        scale = c.dim ** -0.5 if scale is None else scale
        out, lse = ref.decode(got[0], out_t), got[1].astype(np.float64)
        taken = set()
        for r, (first, n) in enumerate(self.runs):
            taken |= set(range(first, first + n))
            total = max(0, min(max([0] + self.lens[first:first + n]), c.max_pages * c.page))
            keys, values = c.tokens(r, range(total)) if total else (np.zeros((0, c.kv, c.dim)),) * 2
            for j in range(first, first + n):
                if j in skip or (rows is not None and j not in rows):
                    continue
                end = max(0, min(self.lens[j], total))
                at = [i for i in range(max(0, end - self.window) if self.window else 0, end) if (r, i) not in hidden]
                o, l, size, dots = ref.attention(self.q[j], keys[at], values[at], scale)
                if not at:
                    assert not out[j].any() and np.all(lse[j] == -np.inf), j
                    continue
                o_tol, l_tol = bounds(o, size, dots, np.abs(values[at]).max() if c.c_t != I8 else 127 * c.scales[1][np.isfinite(c.scales[1])].max(),
                                      c.dim, self.q_t, c.c_t, out_t, len(at))
                l_tol = l_tol + 2.0 ** -22 * np.abs(l)
                for mine, oracle in ((out[j], o), (lse[j], l)):  # a key without a number leaves none, in its head alone
                    assert np.array_equal(np.isnan(mine), np.isnan(oracle)), ("nan", r, j, end, np.isnan(mine).sum(), np.isnan(oracle).sum())
                assert np.all((np.abs(out[j] - o) <= o_tol) | np.isnan(o)), ("out", r, j, end, float(np.nanmax(np.abs(out[j] - o) / o_tol)))
                assert np.all((np.abs(lse[j] - l) <= l_tol) | np.isnan(l)), ("lse", r, j, end, float(np.max(np.abs(lse[j] - l) / l_tol)))
        rest = [j for j in range(self.rows) if j not in taken]
        assert np.all(got[0][rest].view(np.uint8) == 0x5A) and np.all(got[1][rest].view(np.uint8) == 0x5A)


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("q_t,c_t", TYPES)
def test_types_and_dims(qmm, dim, q_t, c_t):
    for out_t in (q_t, F32):
        c = Case(qmm, [0, 5, 0, 70, 300, 0], [1, 40, 0, 3, 70, 130], 8, 2, dim, q_t, c_t, seed=dim + c_t, block=8 if dim == 96 else 16)
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (3, 1), (7, 1), (17, 1), (40, 8), (33, 1), (64, 1), (300, 1), (257, 1), (512, 2)])
def test_head_layouts(qmm, heads, kv_heads):
    for dim, c_t in ((64, I8), (256, BF16)):
        c = Case(qmm, [3, 0], [50, 77], heads, kv_heads, dim, c_t=c_t, seed=heads)
        c.check(c.run(qmm), rows={0, 1, 31, 32, 49, 50, 51, 100, 126})


@pytest.mark.parametrize("block,page", [(8, 8), (8, 24), (8, 40), (16, 64), (32, 160), (32, 256)])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_pages_and_layouts(qmm, block, page, layout):
    c = Case(qmm, [0, 23, 400], [100, 33, 65], 6, 3, 64, block=block, page=page, layout=layout, seed=page, max_pages=1000 // page)
    c.check(c.run(qmm))
    c = Case(qmm, [10, 300], [20, 65], 4, 2, 192, F16, F16, page=page, layout=layout, seed=page)
    c.check(c.run(qmm))


@pytest.mark.parametrize("window", [1, 2, 31, 63, 64, 65, 200])
@pytest.mark.parametrize("c_t", [I8, BF16])
def test_window(qmm, window, c_t):
    c = Case(qmm, [0, 100, 1000], [150, 7, 90], 8, 2, 128, c_t=c_t, window=window, seed=window)
    c.check(c.run(qmm))


@pytest.mark.parametrize("held,new", [([5000], [4]), ([9000, 3, 0], [1, 1, 20]), ([20001], [33]), ([1000, 1000], [5, 1])])
@pytest.mark.parametrize("q_t,c_t,dim", [(BF16, I8, 128), (F16, F16, 64), (F16, I8, 256), (BF16, F8, 96)])
def test_keys_split_between_workgroups(qmm, held, new, q_t, c_t, dim):
    for out_t in (q_t, F32):
        c = Case(qmm, held, new, 8, 2, dim, q_t, c_t, seed=dim + len(new))
        c.check(c.run(qmm, out_t), out_t)
    c = Case(qmm, held, new, 8, 2, dim, q_t, c_t, seed=dim, window=1500)
    c.check(c.run(qmm))


def test_many_runs(qmm):
    """More runs than a wave has lanes, many of them empty or of one token."""
    rng = np.random.default_rng(4)
    new = [int(n) for n in rng.choice([0, 0, 1, 1, 2, 40], 300)]
    c = Case(qmm, [int(n) for n in rng.integers(0, 90, 300)], new, 4, 2, 64, seed=4)
    c.check(c.run(qmm))


def test_long_prompt(qmm):
    """Steps by the hundred: compared at some rows."""
    c = Case(qmm, [37], [2500], 16, 2, 128, seed=5)
    c.check(c.run(qmm), rows={0, 1, 15, 16, 17, 1000, 1023, 1024, 2047, 2498, 2499})
    c = Case(qmm, [0], [1500], 2, 2, 64, F16, F16, seed=6)
    c.check(c.run(qmm, F32), F32, rows={0, 63, 64, 255, 256, 257, 1000, 1499})


@pytest.mark.parametrize("c_t", [I8, F8, BF16])
def test_lengths_of_any_kind(qmm, c_t):
    """Rows that see nothing (a step's refused tokens) between others, lengths that fall, negative ones
    and those past the table."""
    lens = [0] * 20 + [5, 90, 1, 0, 64, 63, 65, 33] + [-7, -2 ** 31, 48, 2 ** 31 - 1, 0]
    c = Case(qmm, [0, 85, 30], [20, 8, 5], 4, 2, 64, c_t=c_t, lens=lens, seed=7, max_pages=6)
    # the third request's table holds 96 keys, of which it has 35
    p = c.c
    for col in range(3, 6):
        p.tables[2, col] = -1
    for b in p.bits:
        b[p.tables[2, 2], 3:] = 1
    p.upload(qmm)
    c.check(c.run(qmm), hidden={(2, i) for i in range(48, 96)})


def test_pages_outside(qmm):
    for c_t in (I8, F16):
        c = Case(qmm, [100, 0, 2100], [30, 64, 9], 8, 2, 128, F16, c_t, seed=10)
        hidden = set()
        for r, col, bad in ((0, 1, -1), (0, 6, 2 ** 31 - 1), (1, 0, c.c.n_pages), (1, 1, -5), (1, 2, -2 ** 31), (1, 3, -1), (2, 70, -1)):
            c.c.tables[r, col] = bad
            hidden |= {(r, i) for i in range(col * 16, col * 16 + 16)}
        c.c.upload(qmm)
        c.check(c.run(qmm), hidden=hidden)
        c.check(c.run(qmm, F32), F32, hidden=hidden)


@pytest.mark.parametrize("q_t,c_t", [(BF16, BF16), (F16, F16), (BF16, I8)])
def test_large_and_negative_scores(qmm, q_t, c_t):
    c = Case(qmm, [0, 200], [60, 70], 8, 2, 64, q_t, c_t, k_size=12.0, seed=13)
    for scale in (1.0, -0.5, 0.0):
        for out_t in (q_t, F32):
            c.check(c.run(qmm, out_t, scale=scale), out_t, scale=scale)


def test_scales_of_all_sizes(qmm):
    c = Case(qmm, [0, 150], [300, 50], 8, 2, 64, seed=11)
    p = c.c
    for i in range(2):
        p.scales[i][p.tables[0, 2], 0, 0] = 0
        p.scales[i][p.tables[0, 3], 0, 1] = 2.0 ** -40
        p.scales[i][p.tables[1, 4], 0] = 0
    p.upload(qmm)
    for out_t in (BF16, F32):
        c.check(c.run(qmm, out_t), out_t)


@pytest.mark.parametrize("q_t,c_t", TYPES)
@pytest.mark.parametrize("dim", [64, 256])
def test_values_without_a_number_behind_a_row(qmm, q_t, c_t, dim):
    """A token whose key and value are NaN or infinite: rows before it do not see it, rows from it on
    have NaN where they read it; in the same steps, and where rows are windowed past it."""
    for bad, window in ((np.nan, 0), (np.inf, 0), (np.nan, 24)):
        c = Case(qmm, [0, 37], [90, 20], 4, 2, dim, q_t, c_t, seed=17, window=window)
        p = c.c
        if c_t == F8 and bad != bad:
            code = 0x7F
        elif c_t == F8:
            continue  # no infinities
        at = 50  # of request 0; in I8 its block, 48 to 63
        page = p.tables[0, at // 16]
        if c_t == I8:
            p.scales[1][page, 0, 0] = bad
        else:
            p.bits[1][page, at % 16, 0, 7] = code if c_t == F8 else ref.encode(np.array([bad]), c_t)[0]
        p.upload(qmm)
        for out_t in (q_t, F32):
            got = c.run(qmm, out_t)
            out = ref.decode(got[0], out_t)
            first = 48 if c_t == I8 else at
            until = 90 if not window else min(90, (64 if c_t == I8 else at + 1) + window - 1)
            seeing = range(first, until)
            c.check(got, out_t, skip=set(seeing))
            for j in seeing:
                assert np.isfinite(out[j, 2:]).all() and not np.isfinite(out[j, :2, 7]).any(), j
                if c_t != I8:
                    assert np.isfinite(np.delete(out[j], 7, -1)).all(), j


def test_keys_without_a_number(qmm):
    """-inf has no weight, a row with nothing else is empty; +inf and NaN make the heads that see them
    NaN, and nobody else."""
    c = Case(qmm, [0, 0, 0], [40, 40, 40], 4, 2, 64, c_t=BF16, seed=14)
    p = c.c
    c.qb = ref.encode(np.abs(c.q) + 0.5, BF16)
    c.q = ref.decode(c.qb, BF16)
    c.queries(qmm)
    for key in range(0, 40, 3):
        p.bits[0][p.tables[0, key // 16], key % 16] = 0xFF80
    for key in range(30):
        p.bits[0][p.tables[1, key // 16], key % 16, 0] = 0xFF80
    p.bits[0][p.tables[2, 1], 1, 1] = 0x7F80  # key 17
    p.upload(qmm)
    for out_t in (BF16, F32):
        got = c.run(qmm, out_t)
        out = ref.decode(got[0], out_t)
        c.check(got, out_t, hidden={(0, i) for i in range(0, 40, 3)}, skip=set(range(40, 80)) | set(range(97, 120)))
        assert not out[40:70, :2].any() and np.all(got[1][40:70, :2] == -np.inf) and np.isfinite(out[40:80]).all()
        assert np.isfinite(out[80:120, :2]).all() and np.isnan(out[97:120, 2:]).all() and np.isfinite(out[80:97]).all()


@pytest.mark.parametrize("q_t,c_t", TYPES)
def test_sinks(qmm, q_t, c_t):
    """A first key far above the others whose value is zero: up to 2^-25 of it for 16-bit outputs, and
    any that fp32 holds for fp32 ones."""
    c = Case(qmm, [700], [6], 4, 1, 64, q_t, c_t, seed=13)
    p = c.c
    c.qb = ref.encode(np.abs(c.q) + 0.5, q_t)
    c.q = ref.decode(c.qb, q_t)
    c.queries(qmm)
    page = int(p.tables[0, 0])
    p.bits[1][page, 0] = 0
    for nats, outs in ((10.0, (q_t, F32)), (17.0, (q_t, F32)), (35.0, (F32,))):
        size = nats / (np.abs(c.q[:6]).sum(-1).mean() * 64 ** -0.5)
        if c_t == I8:
            p.bits[0][page, 0] = 127
            p.scales[0][page, 0] = size / 127
        else:
            p.bits[0][page, 0] = ref.encode(np.full((1, 64), size / p.k_scale), c_t)
        p.upload(qmm)
        for out_t in outs:
            c.check(c.run(qmm, out_t), out_t)


def test_strides(qmm):
    c = Case(qmm, [10, 0], [20, 33], 6, 2, 64, c_t=F16, q_t=F16, seed=15)
    n, row = c.rows, 6 * 64
    wide = np.full((n, row + 40), 0x7E00, np.uint16)
    wide[:, :row] = c.qb.reshape(n, -1)
    dq, do = qmm.DeviceBuffer.from_numpy(wide), qmm.DeviceBuffer(n * (row + 8) * 2)
    do.fill(0x5A)
    dlse = qmm.DeviceBuffer(n * 6 * 4)
    dlse.fill(0x5A)
    attn = qmm.PromptAttention(6, 2, 64, F16)
    print("prompt strided", flush=True)
    attn.run(c.c.cache, dq, do, c.c.d_tables, c.c.max_pages, c.ds, c.dl, n, 2, d_lse=dlse, q_stride=row + 40, out_stride=row + 8)
    got = do.download(np.uint16, (n, row + 8))
    assert np.all(got[:, row:] == 0x5A5A)
    c.check((np.ascontiguousarray(got[:, :row]).reshape(n, 6, 64), dlse.download(np.float32, (n, 6))))


def test_odd_starts(qmm):
    """Rows before the first run stay as they were; starts that fall or lie outside write no row
    that is not there."""
    c = Case(qmm, [0, 0], [30, 30], 4, 2, 64, seed=18)
    first = c.run(qmm)
    c.check(first)
    c.starts = [7, 30, 41]
    c.queries(qmm)
    got = c.run(qmm)
    assert np.all(got[0][:7].view(np.uint8) == 0x5A) and np.all(got[0][41:].view(np.uint8) == 0x5A)
    assert np.array_equal(got[0][7:41], first[0][7:41]) and np.array_equal(got[1][7:41], first[1][7:41])
    for starts in ([-5, 2, 2 ** 31 - 1], [9, 4, 1], [2 ** 31 - 1, -1, -2 ** 31], [0, 0, 0]):
        c.starts = starts
        c.queries(qmm)
        got = c.run(qmm)
        if starts == [0, 0, 0]:
            assert np.all(got[0].view(np.uint8) == 0x5A)


def test_offsets_past_32_bits(qmm):
    page, kv_heads, dim = 256, 8, 128
    for c_t, block in ((I8, 32), (BF16, 16)):
        c = Case(qmm, [600, 0], [20, 40], 16, kv_heads, dim, c_t=c_t, page=page, block=block, seed=16)
        p = c.c
        per_page, per_scales = page * kv_heads * dim * kv.SIZE[c_t], page // block * kv_heads * 4
        n_pages = (9 << 29) // per_page + 2
        d, ds = [qmm.DeviceBuffer(n_pages * per_page) for _ in range(2)], [qmm.DeviceBuffer(n_pages * per_scales) for _ in range(2)]
        shift = n_pages - p.n_pages
        for i in range(2):
            for buf, src, each in ((d[i], p.bits[i], per_page),) + (((ds[i], p.scales[i], per_scales),) if c_t == I8 else ()):
                qmm.stream_copy(kv.at_page(buf, shift * each, src.nbytes), qmm.DeviceBuffer.from_numpy(src), src.nbytes)
        more = dict(block=block, d_k_scales=ds[0], d_v_scales=ds[1]) if c_t == I8 else {}
        p.cache = qmm.KVCache(d[0], d[1], c_t, n_pages, page, kv_heads, dim, **more)
        p.d_tables = qmm.DeviceBuffer.from_numpy(np.where((p.tables >= 0) & (p.tables < p.n_pages), p.tables + shift, -1).astype(np.int32))
        c.check(c.run(qmm))


def test_equal_calls_give_equal_bits(qmm):
    """On another stream, and with a workspace that calls of other sizes used in between."""
    a = Case(qmm, [9000, 0], [3, 40], 16, 2, 128, seed=17)
    b = Case(qmm, [3000], [5], 8, 4, 64, F16, F16, seed=18)
    first_of, second_of = qmm.PromptAttention(16, 2, 128), qmm.PromptAttention(8, 4, 64, F16, F32)
    big = first_of.work if first_of.work.nbytes >= second_of.work.nbytes else second_of.work
    first_of.work = second_of.work = big
    first, second = a.run(qmm, attn=first_of), b.run(qmm, F32, attn=second_of)
    a.check(first)
    b.check(second, F32)
    s = qmm.Stream()
    for i in range(4):
        st = s.handle if i % 2 else None
        for c, at, want, out_t in ((a, first_of, first, BF16), (b, second_of, second, F32)):
            got = c.run(qmm, out_t, attn=at, stream=st)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1].view(np.uint32), want[1].view(np.uint32)), i


def test_graph_replays(qmm):
    """A captured call, replayed with other runs and lengths in its buffers."""
    from openmini_qmm.hip_runtime import Graph
    c = Case(qmm, [2000, 10], [60, 30], 8, 2, 128, seed=19)
    attn, s, n = qmm.PromptAttention(8, 2, 128), qmm.Stream(), 93
    do, dlse = qmm.DeviceBuffer(n * 8 * 128 * 2), qmm.DeviceBuffer(n * 8 * 4)
    g = Graph(s.handle, lambda st: attn.run(c.c.cache, c.dq, do, c.c.d_tables, c.c.max_pages, c.ds, c.dl, n, 2, d_lse=dlse, stream=st))
    for rep, (a, b) in enumerate(((60, 30), (1, 0), (0, 37), (90, 0))):
        c.runs, c.starts = [(0, a), (a, b)], [0, a, a + b]
        c.lens = [1900 + i for i in range(a)] + [2 + i for i in range(b)] + [1] * (n - a - b)
        c.ds.upload(np.array(c.starts, np.int32), s.handle)
        c.dl.upload(np.array(c.lens, np.int32), s.handle)
        do.fill(0x5A, s.handle)
        dlse.fill(0x5A, s.handle)
        print(f"prompt graph replay {rep}", flush=True)
        g.launch(s.handle)
        s.synchronize()
        got = do.download(np.uint16, (n, 8, 128)), dlse.download(np.float32, (n, 8))
        c.check(got)
        assert np.array_equal(c.run(qmm, attn=attn)[0], got[0])


def test_no_rows(qmm):
    c = Case(qmm, [5], [1], 4, 2, 64)
    attn = qmm.PromptAttention(4, 2, 64)
    attn.run(c.c.cache, c.dq, c.dl, c.c.d_tables, 1, c.ds, c.dl, 0, 1)
    with pytest.raises(qmm.QmmError, match="d_out is d_q"):
        attn.run(c.c.cache, c.dq, c.dq, c.c.d_tables, 1, c.ds, c.dl, 1, 1)


@pytest.mark.parametrize("dim", [192, 256])
@pytest.mark.parametrize("q_t,c_t", TYPES)
def test_more_workgroups_than_have_a_cu_each(qmm, dim, q_t, c_t):
    """Wide heads in two workgroups a CU; scores so far apart that what two fp16 parts leave counts, and keys in e4m3 past its largest number: NaN."""
    rng = np.random.default_rng(dim)
    held, new = [int(n) for n in rng.integers(0, 70, 56)], [int(n) for n in rng.integers(1, 4, 56)]
    c = Case(qmm, held, new, 8, 8, dim, q_t, c_t, seed=dim + c_t, k_size=6.0)
    for out_t in (q_t, F32):
        c.check(c.run(qmm, out_t), out_t)
