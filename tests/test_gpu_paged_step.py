"""The paged decoder layer end to end: a sequence in chunks and single tokens gives what one
pass over all of it gives, and the layer's parts agree with 64 bits; the serving loop
returns every page.

Two runs of the same rows differ by the attention's rounding (a different split of the
keys), which can move an int8 token by one step; a step is 1/127 of its chunk's maximum
and one chunk's value in 127 moves at most, so y agrees within 2 % of its row's norm."""
import pytest
import torch

from thunderllamax_b200 import ops, paged, paged_step

pytestmark = pytest.mark.gpu
SMALL = paged_step.LayerShape(heads=4, kv_heads=2, head_dim=128, dim=512, ffn=512)


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.require_device()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("cache", [torch.float16, "int8"])
def test_chunks_agree_with_one_pass(cache):
    n, page = 150, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    q, gate = (torch.randn((n, 4, 128), generator=g, device="cuda").half() for _ in range(2))
    k, v = (torch.randn((n, 2, 128), generator=g, device="cuda").half() for _ in range(2))
    res = torch.randn((n, 512), generator=g, device="cuda")
    layer = paged_step.PagedLayer(n, 12, page, SMALL, cache=cache, seed=3)
    table = paged.PageTable(1, 12, 12, page)
    plan = table.plan(i32([0]), i32([n]), paged.Plan(1, n))
    whole_res = res.clone()
    whole = layer(plan, table.table, q, k, v, whole_res, gate=gate)
    table.release(i32([1]))
    done, ys, rs = 0, [], []
    for step in (64, 40, 1, 1, 17, 26, 1):
        plan = table.plan(i32([done]), i32([step]), paged.Plan(1, step))
        cut = slice(done, done + step)
        r = res[cut].clone()
        ys.append(layer(plan, table.table, q[cut], k[cut], v[cut], r, gate=gate[cut]))
        rs.append(r)
        done += step
    torch.cuda.synchronize()
    assert done == n and layer.errors() == 0
    y, r = torch.cat(ys), torch.cat(rs)
    assert (r - whole_res).norm() <= 2e-3 * whole_res.norm()
    assert ((y - whole).norm(dim=1) <= 0.02 * whole.norm(dim=1)).all()


def test_serving_loop_returns_its_pages():
    prompts, page = [130, 5, 64, 1], 16
    pages = sum(-(-(p + 4) // page) for p in prompts)
    layer = paged_step.PagedLayer(200, pages, page, SMALL)
    steps, tokens = paged_step.serve(layer, prompts, 4, 48, pages, page)
    assert tokens == sum(prompts) + 4 * 4 and steps >= 7


def test_layer_refuses_too_many_rows():
    layer = paged_step.PagedLayer(8, 4, 16, SMALL)
    plan = paged.Plan(1, 9)
    rows = torch.zeros((9, 4, 128), dtype=torch.float16, device="cuda")
    with pytest.raises(ops.TLXError):
        layer(plan, i32([[0, 1, 2, 3]]), rows, rows[:, :2], rows[:, :2], torch.zeros((9, 512), device="cuda"))
