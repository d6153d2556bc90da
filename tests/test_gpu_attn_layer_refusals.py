"""What CachedAttention and PagedAttention refuse: arguments whose buffers are all long enough
and whose results would be those of other tokens."""
import pytest

from attn_ref import F16
from test_gpu_attn_step import DIM, HEADS, HIDDEN, KV, MAX_PAGES, PAGE, Layer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(qmm, orc):
    return Layer(qmm, orc, 0x1100, F16, 1)


@pytest.mark.parametrize("heads,kv,dim", [(HEADS // 2, KV, DIM), (HEADS * 2, KV, DIM), (HEADS, KV * 2, DIM), (HEADS, KV, 128)])
def test_shared_attention_of_other_heads(qmm, layer, heads, kv, dim):
    """Fewer query heads: every size check of a call passes, rows are read at another stride."""
    other = qmm.PagedAttention(heads, kv, dim, F16)
    with pytest.raises(qmm.InvalidInput, match="shared attention has heads"):
        qmm.CachedAttention(layer.weights, qmm.Rope(layer.freq), layer.cache, HEADS, 64, F16, attention=other)
    step = qmm.CachedAttention(layer.weights, qmm.Rope(layer.freq), layer.cache, HEADS, 64, F16,
                               attention=qmm.PagedAttention(HEADS, KV, DIM, F16))
    with pytest.raises(qmm.InvalidInput, match="shared attention has heads"):
        step.attention = other


@pytest.mark.parametrize("page", [8, 32, 64])
def test_plan_of_another_page_size(qmm, layer, page):
    """Its slots and table columns would be other tokens' in the layer's cache."""
    plan = qmm.StepPlan(page, 1, 64, MAX_PAGES)
    d = qmm.DeviceBuffer(1 << 18)
    with pytest.raises(qmm.InvalidInput, match="pages of"):
        layer.step.forward_device(d, plan, d, 1, 3, d)


def test_positions_of_several_axes_are_needed(qmm, orc):
    """The plan's one row of positions is no [axes][tokens], long enough as it may be."""
    layer = Layer(qmm, orc, 0x1200, F16, 3)
    plan = qmm.StepPlan(PAGE, 1, 64, MAX_PAGES)
    d = qmm.DeviceBuffer(1 << 18)
    with pytest.raises(qmm.InvalidInput, match="the rope has 3"):
        layer.step.forward_device(d, plan, d, 1, 3, d)


def test_short_buffers(qmm, layer):
    """The projections write as many rows as they are told."""
    plan = qmm.StepPlan(PAGE, 1, 64, MAX_PAGES)
    d, short = qmm.DeviceBuffer(1 << 18), qmm.DeviceBuffer(3 * HIDDEN * 4 - 4)
    with pytest.raises(qmm.InvalidInput, match="d_x holds"):
        layer.step.forward_device(short, plan, d, 1, 3, d)
    with pytest.raises(qmm.InvalidInput, match="d_out holds"):
        layer.step.forward_device(d, plan, d, 1, 3, short)
