"""What the front ends of the paged-serving operators hand to the library, without a GPU: an
address on the host, or on another GPU than the rest, has to be refused before the call.
Tensors are stand-ins with a device of their own, the library a recorder."""
import pytest
import torch

from thunderllamax_b200 import _lib, ops, prefill

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
