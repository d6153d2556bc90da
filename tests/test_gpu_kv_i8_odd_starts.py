"""Runs whose starts are negative, fall or pass the rows: rows of a run are its tokens, and nothing
behind the call's rows is written (memory there belongs to others)."""
import numpy as np
import pytest

import kv_i8_ref as kv
import test_gpu_attn_prompt as prompt
from attn_ref import BF16, F32

pytestmark = pytest.mark.gpu
I8, GUARD = kv.I8, 16
TOP = 2 ** 31 - 1


@pytest.mark.parametrize("starts", [[-5, 2, TOP], [0, 5, TOP], [3, 3, 8], [9, 4, 1], [TOP, -1, -2 ** 31], [TOP] * 3, [-9, -4, -1], [0, 40, 41]])
@pytest.mark.parametrize("rows", [10, 33])
def test_prompts(qmm, starts, rows):
    """A run's rows are those of its starts that the call has.  Where starts fall, rows that both or
    neither of two runs name hold some run's result or what they held."""
    c = prompt.Case(qmm, [40, 40], [30, 30], 4, 2, 64, c_t=I8, seed=18)
    buf = qmm.DeviceBuffer.from_numpy
    c.lens = [41 + i % 30 for i in range(c.rows)]
    c.queries(qmm)
    c.ds = buf(np.array(starts, np.int32))
    do, dlse = qmm.DeviceBuffer((rows + GUARD) * 4 * 64 * 2), qmm.DeviceBuffer((rows + GUARD) * 4 * 4)
    do.fill(0x5A)
    dlse.fill(0x5A)
    print(f"prompt rows={rows} starts={starts}", flush=True)
    qmm.PromptAttention(4, 2, 64).run(c.c.cache, c.dq, do, c.c.d_tables, c.c.max_pages, c.ds, c.dl, rows, 2, d_lse=dlse)
    got = do.download(np.uint16, (rows + GUARD, 4, 64)), dlse.download(np.float32, (rows + GUARD, 4))
    assert np.all(got[0][rows:] == 0x5A5A) and np.all(got[1][rows:].view(np.uint8) == 0x5A)
    if starts == sorted(starts):
        first = [min(max(s, 0), rows) for s in starts]
        c.rows, c.runs = rows, [(a, b - a) for a, b in zip(first, first[1:])]
        c.check((got[0][:rows], got[1][:rows]))


@pytest.mark.parametrize("starts", [[-5, 2, TOP], [0, 5, TOP], [3, 3, 8], [9, 4, 1], [TOP, -1, -2 ** 31], [TOP] * 3, [-9, -4, -1], [0, 40, 41]])
def test_reading_back(qmm, starts):
    """The first row of a run that starts before row 0 is as many tokens on."""
    c = kv.Paged(qmm, [60, 60], 1, 64, I8, seed=6)
    buf, rows = qmm.DeviceBuffer.from_numpy, 10
    outs = [qmm.DeviceBuffer((rows + GUARD) * 64 * 4) for _ in range(2)]
    for o in outs:
        o.fill(0x5A)
    print(f"read starts={starts}", flush=True)
    c.cache.read(c.d_tables, c.max_pages, buf(np.array(starts, np.int32)), 2, rows, *outs, F32)
    for i, o in enumerate(outs):
        got = o.download(np.uint32, (rows + GUARD, 64))
        assert np.all(got[rows:] == 0x5A5A5A5A)
        if starts != sorted(starts):
            continue
        for j in range(rows):
            mine = [(r, j - a) for r, (a, b) in enumerate(zip(starts, starts[1:])) if a <= j < b]
            if not mine:
                assert np.all(got[j] == 0x5A5A5A5A), j
                continue
            r, t = mine[0]
            page, off = divmod(t, c.page)
            want = c.bits[i][c.tables[r, page], off, 0].astype(np.float32) * c.scales[i][c.tables[r, page], off // c.block, 0]
            assert np.array_equal(got[j], want.view(np.uint32)), (i, j)
