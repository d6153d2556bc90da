"""What a list of free pages that runs out means for the requests behind."""
import pytest

from test_gpu_attn_plan import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_free", range(0, 10))
def test_shortage_refuses_those_behind(qmm, n_free):
    """Needs of 3, 4, 1, 0 and 1 pages: from the first that is short of pages on, all that need some
    are refused, also where what is left would do for them."""
    _run(qmm, [0, 0, 0, 5, 16], [48, 64, 16, 3, 1], 16, 8, n_free, 200)
