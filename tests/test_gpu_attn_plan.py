"""openmini_kv_plan on the GPU against a plain restatement: whole numbers, equal."""
import numpy as np
import pytest

import attn_ref as ref

pytestmark = pytest.mark.gpu
OUT = ("starts", "lens", "rows", "positions", "slots", "row_lens", "counts")


def _run(qmm, cached, new, page, max_pages, n_free, max_tokens, head=None, stride=None, seed=0, stream=None, plan=None):
    rng = np.random.default_rng(seed)
    R, stride = len(cached), stride or max_pages
    order = rng.permutation(1 << 14).astype(np.int32)
    free = order[:n_free]
    tables = np.full((R, stride), -7, np.int32)
    at = n_free
    for r, c in enumerate(cached):
        held = min(-(-max(int(c), 0) // page), max_pages)
        tables[r, :held] = np.resize(order[at:], held)
        at = (at + held) % (len(order) - 1)
    want_tables = tables.copy()
    want = ref.plan(cached, new, free, head or 0, want_tables, max_pages, page, max_tokens)
    buf = qmm.DeviceBuffer.from_numpy
    dt, df = buf(tables), buf(free) if n_free else qmm.DeviceBuffer(4)
    plan = plan or qmm.StepPlan(page, R, max_tokens, max_pages)
    for name in OUT:
        getattr(plan, name).fill(0x55)
    print(f"plan R={R} page={page} pages={max_pages} free={n_free} tokens={sum(max(int(n), 0) for n in new)} of {max_tokens}", flush=True)
    plan.run(buf(np.array(cached, np.int32)), buf(np.array(new, np.int32)), R, dt, df, n_free,
             d_head=buf(np.array([head], np.int32)) if head is not None else None, stream=stream, table_stride=stride)
    for name in OUT:
        got = getattr(plan, name).download(np.int32, want[name].shape, stream)
        assert np.array_equal(got, want[name]), name
    assert np.array_equal(dt.download(np.int32, tables.shape, stream), want_tables)


@pytest.mark.parametrize("page", [1, 7, 16, 256])
@pytest.mark.parametrize("cached,new", [
    ([0], [1]), ([0], [0]), ([15], [1]), ([16], [1]), ([17], [40]), ([0, 3, 31, 32, 33], [1, 0, 2, 1, 100]),
    ([-5, 7], [-3, 4]), ([0] * 9, [0] * 9)])
def test_small(qmm, page, cached, new):
    _run(qmm, cached, new, page, max(2, 160 // page), 400, 150)


@pytest.mark.parametrize("R", [63, 64, 65, 255, 256, 257, 1000, 4096])
def test_many_requests(qmm, R):
    rng = np.random.default_rng(R)
    cached = rng.integers(0, 500, R)
    new = np.where(rng.random(R) < 0.02, rng.integers(1, 400, R), rng.integers(0, 2, R))
    _run(qmm, cached, new, 16, 60, 9000, int(new.sum()) + 11, seed=R)


def test_long_prompts(qmm):
    _run(qmm, [0, 100000, 5], [50000, 30000, 1], 16, 9000, 8000, 80001)


@pytest.mark.parametrize("n_free", [0, 1, 5, 6, 7])
def test_list_runs_out(qmm, n_free):
    # needs 2, 0, 3, 1, 2 pages: refused from some request on, but for those that need none
    _run(qmm, [16, 3, 0, 32, 15], [20, 4, 48, 1, 30], 16, 8, n_free, 120)


def test_head_and_next_head(qmm):
    for head in (-3, 0, 2, 6, 9, 50):
        _run(qmm, [16, 3, 0], [20, 4, 48], 16, 8, 9, 100, head=head)


def test_too_long_for_the_table(qmm):
    # refused without taking pages: those after it get them
    _run(qmm, [60, 0, 2 ** 31 - 1, 10], [5, 10, 2 ** 31 - 1, 10], 16, 4, 30, 64)


def test_more_tokens_than_planned(qmm):
    _run(qmm, [0, 10, 20], [30, 30, 30], 8, 20, 100, 47)
    _run(qmm, [0, 10, 20], [30, 30, 30], 8, 20, 100, 1)


def test_table_stride_and_stream(qmm):
    s = qmm.Stream()
    _run(qmm, [7, 90, 31], [100, 2, 1], 16, 12, 50, 128, stride=19, stream=s.handle)


def test_sums_stop_at_the_largest(qmm):
    most = 2 ** 31 - 1
    _run(qmm, [0, 0, 0, 3], [most, most, 5, 1], 16, 4, 30, 20)


def test_graph_replays(qmm):
    """A captured step, replayed with other lengths in its buffers."""
    from openmini_qmm.hip_runtime import Graph
    R, page, mp, T = 5, 16, 10, 200
    s = qmm.Stream()
    dc, dn = qmm.DeviceBuffer(4 * R), qmm.DeviceBuffer(4 * R)
    free = np.arange(50, 0, -1).astype(np.int32)
    df, dt = qmm.DeviceBuffer.from_numpy(free), qmm.DeviceBuffer(4 * R * mp)
    plan = qmm.StepPlan(page, R, T, mp)
    g = Graph(s.handle, lambda st: plan.run(dc, dn, R, dt, df, 50, stream=st))
    rng = np.random.default_rng(5)
    for rep in range(4):
        cached, new = rng.integers(0, 60, R), rng.integers(0, 40, R)
        tables = np.arange(R * mp).reshape(R, mp).astype(np.int32)
        dc.upload(cached.astype(np.int32), s.handle)
        dn.upload(new.astype(np.int32), s.handle)
        dt.upload(tables, s.handle)
        print(f"plan graph replay {rep}", flush=True)
        g.launch(s.handle)
        s.synchronize()
        want = ref.plan(cached, new, free, 0, tables, mp, page, T)
        for name in OUT:
            assert np.array_equal(getattr(plan, name).download(np.int32, want[name].shape), want[name]), name
        assert np.array_equal(dt.download(np.int32, tables.shape), tables)
