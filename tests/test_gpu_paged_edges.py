"""Paged attention at the edges of what its header promises."""
import pytest
import torch

from test_gpu_paged import BF16, F16, Batch, device  # noqa: F401
from thunderllamax_b200 import paged

pytestmark = pytest.mark.gpu
CACHES = [F16, BF16, "int8"]


# ------------------------------------------------------------- fewer rows than planned
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,max_new", [([3, 1], 1), ([7, 2], 3), ([60, 1], 20), ([150, 40], 40)])
def test_rows_past_max_new_change_nothing(hd, cache, new, max_new):
    # rows past max_new are not written, and the K and V of those tokens reach no row
    b = Batch(new, [n + 70 for n in new], 4, 2, hd, cache, 16, seed=3, stale=False)
    attn = paged.PagedAttention(4, 2, hd)

    def run():
        out = torch.full_like(b.q, 7.0)
        return attn(b.store, b.table, b.q_start, b.kv_len, b.q, out=out, max_new=max_new)

    clean = run()
    for r, n in enumerate(new):
        for i in range(min(n, max_new) + 70, n + 70):          # tokens of rows that are not asked for
            page, off = int(b.table[r, i // 16]), i % 16
            if cache == "int8":
                b.store.k_scale[page, :, off] = float("nan")
                b.store.v_scale[page, 0, off] = float("inf")
                b.store.v_scale[page, 1, off] = float("nan")
            else:
                b.store.k[page, :, off] = float("nan")
                b.store.v[page, 0, off, 3] = float("inf")
                b.store.v[page, 1, off] = float("nan")
    got = run()
    assert torch.equal(got, clean)
    at = 0
    for n in new:
        m = min(n, max_new)
        assert got[at:at + m].isfinite().all() and (got[at + m:at + n] == 7).all()
        at += n
    assert attn.error() == 0


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


# ------------------------------------------------------------------------- the gate's ends
@pytest.mark.parametrize("cache,hd", [(F16, 64), (BF16, 128), (F16, 256), (BF16, 256)])
@pytest.mark.parametrize("n,kv", [(1, 50), (1, 9000), (40, 90), (40, 9000)])
def test_gate_far_below_zero(cache, hd, n, kv):
    # sigmoid(-88) is 6e-39: an infinite value stays infinite under it, a large one does not vanish
    b = Batch([n], [kv], 4, 2, hd, cache, 16, seed=2, gate=True, stale=False)
    b.gate.fill_(-88.0)
    page = int(b.table[0, 0])
    b.store.v[page, :, 0, 5] = float("inf")
    got = b.attend()
    assert (got[..., 5] == float("inf")).all()
    if cache == BF16:
        b.store.v.fill_(2.0 ** 60)
        want = 2.0 ** 60 * torch.sigmoid(torch.tensor(-88.0, dtype=torch.float64)).item()
        # (the fast exponential is within 2^-16 of its value at 88)
        assert ((b.attend().double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -15)).all()
