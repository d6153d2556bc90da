"""Caches of 4 GiB and more under tables so wide that rows are cut, in the forms that are not read
past the caches: heads that share lines, caches that begin inside one, more query heads to a
key head than a tile has, and calls of too few keys for it."""
import ctypes

import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F8
from test_gpu_attn_decode import Case

pytestmark = pytest.mark.gpu
PAGE = 256


@pytest.mark.parametrize("dim,heads,kv,q_t,c_t,shift,max_pages", [
    (96, 16, 8, BF16, BF16, 0, 64), (96, 16, 8, F16, F16, 0, 64), (96, 16, 8, F16, F8, 0, 64), (128, 16, 8, BF16, BF16, 16, 64),
    (64, 16, 8, F16, F16, 16, 64), (192, 4, 4, F16, F16, 64, 64), (256, 4, 4, BF16, F8, 16, 64), (128, 64, 2, BF16, BF16, 0, 64),
    (128, 16, 8, BF16, BF16, 0, 20), (256, 8, 4, F16, F16, 0, 9)])
def test_offsets_past_32_bits(qmm, dim, heads, kv, q_t, c_t, shift, max_pages):
    """Pages more than 4 GiB into the cache, some of them before it."""
    per_page = PAGE * kv * dim * ref.SIZE[c_t]
    n_pages = (9 << 29) // per_page + 2  # 4.5 GiB
    c = Case(qmm, [600, 2200, 1], heads, kv, dim, q_t, c_t, page=PAGE, seed=dim + shift, max_pages=max_pages)
    # every other page of the case in the last GiB, the others where they were
    far = n_pages - c.n_pages
    inside = (c.tables >= 0) & (c.tables < c.n_pages)
    to = np.arange(c.n_pages) + far * (np.arange(c.n_pages) % 2)
    d = qmm.DeviceBuffer((n_pages + 64) * per_page + shift)  # values from page 0 on, keys from page 64 on
    d_v, d_k = d.ptr.value + shift, d.ptr.value + shift + 64 * per_page
    print(f"attn over {n_pages * per_page} bytes, heads {heads}/{kv} of {dim}, q {q_t} cache {c_t}, shift {shift}, {max_pages} pages", flush=True)
    # where keys and values share pages of the buffer, none of the case's are
    used = {int(t) for t in to} | {int(t) + 64 for t in to}
    assert c.n_pages <= 64 and len(used) == 2 * c.n_pages
    for base, bits in ((d_k, c.kb), (d_v, c.vb)):
        for p in range(c.n_pages):
            at = type("At", (), dict(ptr=ctypes.c_void_p(base + int(to[p]) * per_page), nbytes=per_page))
            qmm.stream_copy(at, qmm.DeviceBuffer.from_numpy(bits[p:p + 1]), per_page)
    cache = qmm.KVCache(d, d, c_t, n_pages, PAGE, kv, dim, k_scale=c.k_scale, v_scale=c.v_scale)
    cache.desc.d_k, cache.desc.d_v = ctypes.c_void_p(d_k), ctypes.c_void_p(d_v)
    dt = qmm.DeviceBuffer.from_numpy(np.where(inside, to[np.where(inside, c.tables, 0)], -1).astype(np.int32))
    do, dlse = qmm.DeviceBuffer(3 * heads * dim * 4), qmm.DeviceBuffer(3 * heads * 4)
    qmm.PagedAttention(heads, kv, dim, q_t).run(cache, c.dq, do, dt, c.max_pages, c.dl, 3, d_lse=dlse)
    c.check((do.download(np.uint32, (3, heads, dim)), dlse.download(np.float32, (3, heads))))
