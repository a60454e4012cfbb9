"""Paged attention at the edges of what its header promises."""
import pytest
import torch

from test_gpu_paged import BF16, F16, Batch, device  # noqa: F401

pytestmark = pytest.mark.gpu
CACHES = [F16, BF16, "int8"]


# ----------------------------------------------------------------- weights that sum to one
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,kv", [(1, 900), (8, 900), (64, 900), (64, 40000)])
def test_equal_values_come_out_as_they_are(hd, cache, n, kv):
    # of every 64 keys one lies above the others, which have one weight each row: rounding that
    # weight moves the sum of the products and has to move the sum of the weights alike.  With
    # V = 1 everywhere every row is 1: fp32 sums of up to 40000 terms are within 2^-13 of it, less
    # than half a step.
    b = Batch([n], [kv], 4, 2, hd, cache, 16, seed=1, stale=False)
    tops = b.table[0, : -(-kv // 16) : 4].long()               # the pages that start a unit
    if cache == "int8":
        b.store.k.fill_(128)
        b.store.k_scale.fill_(1.0 / 64)
        b.store.k[tops, :, 0] = 192                            # 1.0
        b.store.v.fill_(192)
        b.store.v_scale.fill_(1.0 / 64)
    else:
        b.store.k.zero_()
        b.store.k[tops, :, 0] = 1.0
        b.store.v.fill_(1.0)
    length = torch.linspace(0.2, 1.5, n * 4, device="cuda").view(n, 4, 1)   # scores, in nats
    b.q.copy_((length * hd ** -0.5).expand(n, 4, hd).to(b.dtype))
    got = b.attend()
    assert (got == 1).all(), (got - 1).abs().max()
