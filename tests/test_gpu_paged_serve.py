"""The serving loop with no more pages than its running requests need."""
import pytest

from test_gpu_paged_step import SMALL, device  # noqa: F401
from thunderllamax_b200 import ops, paged_step

pytestmark = pytest.mark.gpu


def test_finished_requests_take_no_pages():
    # the short request is done long before the long one needs the pool's last page
    layer = paged_step.PagedLayer(20, 7, 16, SMALL)
    steps, tokens = paged_step.serve(layer, [100, 1], 1, 10, 7, 16)
    assert (steps, tokens) == (11, 103)


def test_a_pool_that_is_too_small_is_refused():
    layer = paged_step.PagedLayer(20, 6, 16, SMALL)
    with pytest.raises(ops.TLXError):
        paged_step.serve(layer, [100, 1], 1, 10, 6, 16)
