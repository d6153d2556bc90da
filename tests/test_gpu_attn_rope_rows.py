"""Rotary positions and the cache write where tokens share a workgroup: few and many heads to
a token, numbers of tokens that do not divide a workgroup's, calls short and long enough for
either form.  Bounds as in test_gpu_attn_rope."""
import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8
from test_gpu_attn_rope import _append, _close, _freq, _inputs, _size

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("xt,yt", [(F32, BF16), (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("tokens,heads,dim,pairs", [
    (31, 1, 8, 4), (33, 1, 8, 4), (65700, 1, 8, 4), (10, 3, 64, 32), (11, 3, 64, 32), (21, 3, 64, 20), (21001, 3, 64, 32),
    (2051, 16, 128, 64), (4099, 15, 128, 64), (4099, 17, 128, 64), (1031, 33, 128, 48), (5003, 5, 96, 48)])
def test_apply_rows(qmm, xt, yt, tokens, heads, dim, pairs):
    rng = np.random.default_rng(tokens + heads)
    print(f"rope {tokens} x {heads} x {dim}, {pairs} pairs {xt}->{yt}", flush=True)
    bits, x = _inputs(rng, (tokens, heads, dim), xt)
    pos = rng.integers(0, 40000, (2, tokens)).astype(np.int32)
    axis = [i % 2 for i in range(pairs)]
    guard = 64
    dy = qmm.DeviceBuffer(x.size * ref.SIZE[yt] + guard)
    dy.fill(0x5A)
    qmm.Rope(_freq(pairs), axes=axis).apply(qmm.DeviceBuffer.from_numpy(bits), xt, dy, yt, qmm.DeviceBuffer.from_numpy(pos), tokens, heads, dim)
    raw = dy.download(np.uint8, (x.size * ref.SIZE[yt] + guard,))
    got = ref.decode(raw[:-guard].view(ref.BITS[yt]).reshape(x.shape), yt)
    _close(got, ref.rope(x, pos, _freq(pairs), axis), _size(x, pairs, False), yt)
    assert np.all(raw[-guard:] == 0x5A)


@pytest.mark.parametrize("in_t,q_t,c_t,layout", [(F32, BF16, BF16, "head"), (F32, F16, F8, "token"), (BF16, BF16, BF16, "token")])
@pytest.mark.parametrize("tokens,heads,kv,dim,pairs", [(13, 1, 1, 16, 8), (4099, 1, 1, 64, 32), (12007, 2, 1, 64, 16), (2053, 12, 4, 128, 64)])
def test_append_rows(qmm, in_t, q_t, c_t, layout, tokens, heads, kv, dim, pairs):
    rng = np.random.default_rng(tokens)
    n_pages = tokens // 16 + 3
    slots = rng.permutation(n_pages * 16)[:tokens].astype(np.int32)
    slots[rng.random(tokens) < 0.05] = -1
    _append(qmm, rng, tokens, heads, kv, dim, pairs, 1, in_t, q_t, c_t, 16, layout, slots, n_pages)
