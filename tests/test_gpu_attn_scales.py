"""Scales of a cache at the ends of fp32."""
import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F32

pytestmark = pytest.mark.gpu


def _append(qmm, x, k_scale, v_scale):
    cache = qmm.KVCache.allocate(BF16, 1, 8, 1, 8, k_scale=k_scale, v_scale=v_scale)
    buf = qmm.DeviceBuffer.from_numpy
    d, zero = buf(x.astype(np.float32)), buf(np.zeros(1, np.int32))
    qmm.Rope([1.0] * 4).append(cache, d, d, d, F32, qmm.DeviceBuffer(16), BF16, zero, zero, 1, 1)
    return [ref.decode(b.download(np.uint16, (64,))[:8], BF16) for b in (cache.d_k, cache.d_v)]


@pytest.mark.parametrize("k_scale,v_scale", [(1e-39, 1.0), (1.0, 1e-39), (2.0 ** -128, 1.0)])
def test_scales_without_a_reciprocal(qmm, k_scale, v_scale):
    """1 / scale is infinite: a zero would be stored as NaN."""
    with pytest.raises(qmm.QmmError, match="reciprocal"):
        _append(qmm, np.zeros(8), k_scale, v_scale)


@pytest.mark.parametrize("scale", [2.0 ** -127, 2.0 ** -126, 3e38])
def test_scales_at_the_ends(qmm, scale):
    """Numbers of the scale's size become their quotients: the reciprocal of 3e38 is a subnormal of
    22 bits, and bf16 rounds to 8."""
    x = np.array([0, 1, -1, 0.5, 0.75, -0.25, 0, 1]) * scale
    for got in _append(qmm, x, scale, scale):
        want = np.float64(x.astype(np.float32)) / np.float64(np.float32(scale))
        assert np.all(np.abs(got - want) <= (2.0 ** -8 + 2.0 ** -20) * np.abs(want)), (got, want)
