"""What the front ends of the paged-serving operators hand to the library, without a GPU: an
address on the host, or on another GPU than the rest, has to be refused before the call.
Tensors are stand-ins with a device of their own, the library a recorder."""
import pytest
import torch

from thunderllamax_b200 import _lib, ops, paged, prefill

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class Standin:
    """A host tensor that says it lies on `device`."""

    def __init__(self, t, device="cuda:0"):
        self.t, self.device = t, torch.device(device)

    def __getattr__(self, name):            # shape, dtype, stride, numel, is_contiguous, data_ptr, dim
        return getattr(self.t, name)

    @property
    def is_cuda(self):
        return self.device.type == "cuda"

    def get_device(self):
        return self.device.index


class Library:
    """Counts the calls; every entry point succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 256 if name.endswith("_bytes") else 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "require_device", lambda: None)
    monkeypatch.setattr(ops, "_raw_stream", lambda t: 0)
    return lib


def tensor(shape, dtype, device="cuda:0"):
    return Standin(torch.zeros(shape, dtype=dtype), device)


# ------------------------------------------------------------------------- the norm
def norm_args(**devices):
    at = lambda name: devices.get(name, "cuda:0")
    return dict(x=tensor((4, 256), F32, at("x")), residual=tensor((4, 256), F16, at("residual")),
                weight=tensor((256,), F32, at("weight")), out=tensor((4, 256), F16, at("out")),
                xq=tensor((4, 256), torch.int8, at("xq")), sx=tensor((4, 2), F32, at("sx")),
                rs=tensor((4, 2), torch.int32, at("rs")))


def test_norm_takes_one_device(library):
    prefill.add_rms_norm_q8(**norm_args())
    assert library.calls == ["tlx_add_rms_norm_q8"]


@pytest.mark.parametrize("name", ["x", "residual", "weight", "out", "xq", "sx", "rs"])
@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
def test_norm_refuses_another_device(library, name, where):
    with pytest.raises(_lib.TLXError):
        prefill.add_rms_norm_q8(**norm_args(**{name: where}))
    assert library.calls == []


# ------------------------------------------------------------ plan, release, append, attention
@pytest.fixture
def workspaces(monkeypatch):
    class Space:
        def __init__(self, nbytes, device="cuda"):
            self.nbytes, self.buf = nbytes, tensor((8,), torch.uint8, torch.device(device).type + ":0")

    monkeypatch.setattr(ops, "Workspace", Space)


def i32(n, device="cuda:0"):
    return tensor((n,), torch.int32, device)


def table_of(device="cuda:0", **devices):
    at = lambda name: devices.get(name, device)
    return paged.PageTable(2, 4, 8, 16, table=tensor((2, 4), torch.int32, at("table")), held=i32(2, at("held")),
                           free=i32(8, at("free")), n_free=i32(1, at("n_free")))


class PlanOf:
    def __init__(self, **devices):
        at = lambda name: devices.get(name, "cuda:0")
        self.requests, self.tokens = 2, 3
        for name, n in (("q_start", 3), ("kv_len", 2), ("status", 2), ("slots", 3), ("positions", 3)):
            setattr(self, name, i32(n, at(name)))


def cache_of(**devices):
    at = lambda name: devices.get(name, "cuda:0")
    rows, scales = (8, 2, 16, 64), (8, 2, 16, 2)
    return paged.PagedCache(tensor(rows, torch.uint8, at("k")), tensor(rows, torch.uint8, at("v")),
                            tensor(scales, F16, at("ks")), tensor(scales, F16, at("vs")))


OTHERS = ["cpu", "cuda:1"]


@pytest.mark.parametrize("where", OTHERS)
def test_table_refuses_another_device(library, workspaces, where):
    table_of()
    for name in ("held", "free", "n_free"):
        with pytest.raises(_lib.TLXError):
            table_of(**{name: where})


@pytest.mark.parametrize("where", OTHERS)
def test_plan_refuses_another_device(library, workspaces, where):
    t = table_of()
    t.plan(i32(2), i32(2), PlanOf(), held_out=i32(2), n_free_out=i32(1))
    assert library.calls[-1] == "tlx_paged_plan"
    n = len(library.calls)
    bad = [((i32(2, where), i32(2), PlanOf()), {}), ((i32(2), i32(2, where), PlanOf()), {}),
           ((i32(2), i32(2), PlanOf()), dict(held_out=i32(2, where))),
           ((i32(2), i32(2), PlanOf()), dict(n_free_out=i32(1, where)))]
    bad += [((i32(2), i32(2), PlanOf(**{name: where})), {}) for name in ("q_start", "kv_len", "status", "slots",
                                                                         "positions")]
    for args, kw in bad:
        with pytest.raises(_lib.TLXError):
            t.plan(*args, **kw)
    with pytest.raises(_lib.TLXError):
        t.release(i32(2, where))
    assert len(library.calls) == n


@pytest.mark.parametrize("where", OTHERS)
def test_append_refuses_another_device(library, where):
    c, rows = cache_of(), (3, 2, 64)
    good = dict(k=tensor(rows, F16), v=tensor(rows, F16), slots=i32(3))
    c.append(**good)
    for name, t in (("k", tensor(rows, F16, where)), ("v", tensor(rows, F16, where)), ("slots", i32(3, where))):
        with pytest.raises(_lib.TLXError):
            c.append(**{**good, name: t})
    for name in ("v", "ks", "vs"):
        with pytest.raises(_lib.TLXError):
            cache_of(**{name: where})
    assert library.calls == ["tlx_paged_append"]


@pytest.mark.parametrize("where", OTHERS)
def test_attention_refuses_another_device(library, workspaces, where):
    a, c, rows = paged.PagedAttention(4, 2, 64), cache_of(), (3, 4, 64)
    good = dict(table=tensor((2, 4), torch.int32), q_start=i32(3), kv_len=i32(2), q=tensor(rows, F16),
                gate=tensor(rows, F16), out=tensor(rows, F16))
    a(c, **good)
    n = len(library.calls)
    assert library.calls[-1] == "tlx_paged_attention"
    for name, t in good.items():
        with pytest.raises(_lib.TLXError):
            a(c, **{**good, name: Standin(t.t, where)})
    with pytest.raises(_lib.TLXError):                       # a workspace of another device
        a.ws.buf.device = torch.device(where)
        a(c, **good)
    assert len(library.calls) == n


# ------------------------------------------------------------------------ the current device
def test_calls_need_the_current_device(monkeypatch):
    # the default stream's handle is the same on every device: a call with another device current
    # would launch there, on addresses of the tensors' device
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0x100 + d, raising=False)
    assert ops._raw_stream(tensor((1,), F32)) == 0x100
    with pytest.raises(_lib.TLXError):
        ops._raw_stream(tensor((1,), F32, "cuda:1"))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    assert ops._raw_stream(tensor((1,), F32, "cuda:1")) == 0x101
