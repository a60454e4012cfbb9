"""Paged attention where the running maximum keeps growing along the keys, so that the rows
rescale their sums again and again: the instances of the tiles form with two softmax groups
(head dim 256, and int8 at every head dim), which hand the rows' maxima to each other.

The keys are a staircase along one sign vector: unit by unit of 64 keys the scores stay or
jump by 8.5 to 13 in log2, rows have queries of different length, so that the rows of a tile
rescale at different units, and V falls as the scores grow, so that early keys still count.

Tolerance: the one of test_gpu_paged.py, whose part for the scores (2^-13 where the sum of
|q||k| scale is below 32) grows in proportion to that sum: 2^-18 S, twice in a quotient."""
import math

import pytest
import torch

from test_gpu_paged import BF16, F16, Batch, device  # noqa: F401
from thunderllamax_b200 import paged

pytestmark = pytest.mark.gpu
TWO_GROUPS = [(256, F16), (256, BF16), (256, "int8"), (128, "int8"), (64, "int8")]


class Growing(Batch):
    def __init__(self, new, kv, heads, kv_heads, hd, cache, page, seed, jumps, v_range):
        super().__init__(new, kv, heads, kv_heads, hd, cache, page, seed=seed, stale=False)
        g = torch.Generator(device="cuda").manual_seed(seed + 97)
        sign = torch.where(torch.rand(hd, generator=g, device="cuda") < 0.5, -1.0, 1.0)
        self.score_sum = 0.0
        for b, t in enumerate(kv):
            units = -(-t // 64)
            up = torch.rand(units, generator=g, device="cuda") < jumps
            step = torch.where(up, 8.5 + 4.5 * torch.rand(units, generator=g, device="cuda"), 0.0)
            level = step.cumsum(0)
            level = level - level[-1] / 2                                       # log2, for the longest queries
            fall = (level[-1] - level).clamp(max=v_range)                       # V's exponent
            key = torch.arange(t, device="cuda")
            score = level[key // 64] * math.log(2) + 2 * torch.rand(t, generator=g, device="cuda") - 1
            size = score / math.sqrt(hd)                                        # of a key's elements
            ids = self.table[b, key // page].long()
            for c, sc, amount in ((self.store.k, self.store.k_scale, size),
                                  (self.store.v, self.store.v_scale, torch.exp2(fall[key // 64]))):
                shape = (t, kv_heads, hd)
                noise = torch.rand(shape, generator=g, device="cuda") - 0.5
                is_k = c is self.store.k
                if cache == "int8":
                    way = torch.sign(amount)[:, None, None] * sign if is_k else torch.sign(noise)
                    code = way * 100 + 50 * noise if is_k else 240 * noise
                    c[ids, :, key % page] = (code.round().clamp(-127, 127) + 128).to(torch.uint8)
                    sc[ids, :, key % page] = (amount.abs() / 100).half()[:, None, None].expand(t, kv_heads, hd // 32)
                else:
                    x = amount[:, None, None] * sign + 0.1 * noise if is_k else amount[:, None, None] * 2 * noise
                    c[ids, :, key % page] = x.to(c.dtype)
            self.score_sum = max(self.score_sum, 1.3 * float(score.abs().max()) + 1)
        length = 0.5 + 0.5 * torch.rand(self.q.shape[:2], generator=g, device="cuda")
        self.q.copy_((length[..., None] * sign).to(self.dtype))

    def reference(self):
        ref, tol = super().reference()
        u = 2.0 ** -11 if self.dtype == F16 else 2.0 ** -8
        weight = (tol - 2.0 ** -24 - u * ref.abs()) / (2 * u + 2.0 ** -12)      # sum_j p_j |v_j|
        return ref, tol + 2 * self.score_sum * 2.0 ** -18 * weight

    def check_calls(self, calls):
        attn = paged.PagedAttention(self.heads, self.kv_heads, self.hd)
        ref, tol = self.reference()
        first = None
        for i in range(calls):
            got = attn(self.store, self.table, self.q_start, self.kv_len, self.q, max_new=max(self.new))
            if first is None:
                first = got
                bad = ((got.double() - ref).abs() <= tol).logical_not()
                assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
            assert torch.equal(got.view(torch.int16), first.view(torch.int16)), i
        assert attn.error() == 0


def v_range(cache):
    return 60 if cache == BF16 else 12


@pytest.mark.parametrize("hd,cache", TWO_GROUPS)
@pytest.mark.parametrize("rows", [17, 66, 4096])
def test_long_items_rescale_again_and_again(hd, cache, rows):
    if rows == 4096:
        b = Growing([2048], [8192], 4, 2, hd, cache, 64, rows, 0.25, v_range(cache))
    else:
        b = Growing([rows] * 6, [8192, 8191, 8250, 9001, 8129, 8300], 8, 8, hd, cache, 64, rows, 0.25, v_range(cache))
    b.check_calls(50)


@pytest.mark.parametrize("hd,cache", TWO_GROUPS)
@pytest.mark.parametrize("jumps", [0.3, 0.6, 1.0])
def test_short_items_rescale_in_their_last_units(hd, cache, jumps):
    new = [17 + 7 * i % 50 for i in range(160)]
    kv = [max(n, 256 + 37 * i % 600) for i, n in enumerate(new)]
    Growing(new, kv, 4, 4, hd, cache, 16, int(10 * jumps), jumps, v_range(cache)).check_calls(50)
