"""Argument checks of the paged-serving entry points: every refusal returns its code from
the host before anything is launched, so they run without a GPU."""
import ctypes

import pytest

from thunderllamax_b200 import _lib

P = 0x10000                      # an aligned address that is never read
OK, SHAPE, ALIGN, DTYPE, WORKSPACE, NULL = 0, -1, -2, -3, -5, -8
F32, F16, BF16, Q8 = 0, 1, 30, 102


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def cache(**kw):
    a = dict(k=P, v=P, ks=None, vs=None, stride=(64 * 128 * 2, 64 * 128, 128), sstride=(0, 0, 0), pages=10, page=64,
             heads=2, hd=128, dt=F16)
    a.update(kw)
    return _lib.PagedKV(a["k"], a["v"], a["ks"], a["vs"], a["stride"], a["stride"], a["sstride"], a["sstride"],
                        a["pages"], a["page"], a["heads"], a["hd"], a["dt"])


BAD_CACHES = [(dict(k=None), NULL), (dict(dt=F32), DTYPE), (dict(dt=Q8), NULL), (dict(hd=96), SHAPE),
              (dict(page=24), SHAPE), (dict(page=4), SHAPE), (dict(page=2048), SHAPE), (dict(pages=0), SHAPE),
              (dict(pages=1 << 30), SHAPE), (dict(heads=0), SHAPE), (dict(k=P + 2), ALIGN),
              (dict(stride=(64 * 128 * 2, 64 * 128, 129)), ALIGN), (dict(stride=(-8, 8, 128)), SHAPE),
              (dict(stride=(64 * 128 * 2, 0, 128)), SHAPE), (dict(stride=(1 << 40, 64 * 128, 128)), SHAPE),
              (dict(dt=Q8, ks=P, vs=P, sstride=(512, 0, 4)), SHAPE),
              (dict(dt=Q8, ks=P + 2, vs=P, sstride=(512, 256, 4)), ALIGN),
              (dict(dt=Q8, ks=P, vs=P, sstride=(512, 255, 4)), ALIGN)]


def attention(lib, c, **kw):
    a = dict(table=P, ld=8, width=8, q_start=P, kv=P, n_req=2, q=P, dt=F16, qt=512, qh=128, heads=4, tokens=3, most=3,
             scale=0.1, gate=None, gt=0, gh=0, out=P, ot=512, oh=128, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return lib.tlx_paged_attention(ctypes.byref(c) if c is not None else None, a["table"], a["ld"], a["width"],
                                   a["q_start"], a["kv"], a["n_req"], a["q"], a["dt"], a["qt"], a["qh"], a["heads"],
                                   a["tokens"], a["most"], a["scale"], a["gate"], a["gt"], a["gh"], a["out"], a["ot"],
                                   a["oh"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_cache_refusals(lib, kw, code):
    c = cache(**kw)
    assert attention(lib, c) == code
    assert lib.tlx_paged_append(ctypes.byref(c), P, P, F16, 256, 128, 256, 128, P, 1, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(heads=5), SHAPE), (dict(heads=258), SHAPE), (dict(heads=0), SHAPE), (dict(n_req=0), SHAPE),
    (dict(tokens=-1), SHAPE), (dict(most=-1), SHAPE), (dict(width=0), SHAPE), (dict(ld=7), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(scale=0.0), SHAPE), (dict(scale=-0.1), SHAPE), (dict(scale=float("inf")), SHAPE),
    (dict(dt=F32), DTYPE), (dict(dt=BF16), DTYPE), (dict(table=None), NULL),
    (dict(q_start=None), NULL), (dict(kv=None), NULL), (dict(q=None), NULL), (dict(out=None), NULL),
    (dict(ws=None), NULL), (dict(q=P + 2), ALIGN), (dict(qt=513), ALIGN), (dict(oh=129), ALIGN), (dict(ws=P + 16), ALIGN),
    (dict(gate=P + 8), ALIGN), (dict(gate=P, gt=4), ALIGN), (dict(ws_bytes=8), WORKSPACE), (dict(tokens=0), OK),
    (dict(most=0), OK)])
def test_attention_refusals(lib, kw, code):
    assert attention(lib, cache(), **kw) == code


def test_attention_dtypes(lib):
    assert attention(lib, None) == NULL
    assert attention(lib, cache(dt=BF16), dt=F16) == DTYPE
    assert attention(lib, cache(dt=Q8, ks=P, vs=P, sstride=(512, 256, 4)), dt=BF16) == DTYPE
    assert lib.tlx_paged_attention_workspace_bytes(24, 4, 256) > 0
    for bad in ((5, 4, 256), (24, 4, 100), (0, 1, 64), (4, 0, 64), (129, 1, 64)):
        assert lib.tlx_paged_attention_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(dt=2), DTYPE), (dict(dt=BF16), DTYPE), (dict(n=-1), SHAPE), (dict(n=0), OK), (dict(k=None), NULL),
    (dict(slots=None), NULL), (dict(k=P + 8), ALIGN), (dict(t=257), ALIGN), (dict(h=4), ALIGN),
    (dict(dt=F32, t=130), ALIGN)])
def test_append_refusals(lib, kw, code):
    a = dict(k=P, dt=F16, t=256, h=128, slots=P, n=1)
    a.update(kw)
    c = cache()
    assert lib.tlx_paged_append(ctypes.byref(c), a["k"], P, a["dt"], a["t"], a["h"], 256, 128, a["slots"], a["n"],
                                None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(cached=None), NULL), (dict(slots=None), NULL), (dict(ws=None), NULL), (dict(n_req=0), SHAPE),
    (dict(page=12), SHAPE), (dict(page=4), SHAPE), (dict(width=0), SHAPE), (dict(ld=3), SHAPE), (dict(pages=0), SHAPE),
    (dict(pages=1 << 29), SHAPE), (dict(tokens=-1), SHAPE), (dict(ws=P + 2), ALIGN), (dict(ws_bytes=8), WORKSPACE)])
def test_plan_refusals(lib, kw, code):
    a = dict(cached=P, n_req=2, page=16, ld=4, width=4, pages=9, tokens=3, slots=P, ws=P, ws_bytes=256)
    a.update(kw)
    assert lib.tlx_paged_plan(a["cached"], P, a["n_req"], a["page"], P, a["ld"], a["width"], P, P, P, a["pages"], P, P,
                              a["tokens"], P, P, a["slots"], P, P, a["ws"], a["ws_bytes"], None) == code


def test_release_refusals(lib):
    assert lib.tlx_paged_release(None, 2, P, 4, 4, P, P, 9, P, None) == NULL
    assert lib.tlx_paged_release(P, 0, P, 4, 4, P, P, 9, P, None) == SHAPE
    assert lib.tlx_paged_release(P, 2, P, 3, 4, P, P, 9, P, None) == SHAPE


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), NULL), (dict(sx=None), NULL), (dict(xdt=2), DTYPE), (dict(rdt=102), DTYPE), (dict(m=0), SHAPE),
    (dict(k=200), SHAPE), (dict(k=0), SHAPE), (dict(k=32896), SHAPE), (dict(eps=-1.0), SHAPE),
    (dict(eps=float("nan")), SHAPE), (dict(ldx=100), SHAPE), (dict(ldr=100), SHAPE), (dict(ldh=100), SHAPE),
    (dict(ldq=100), SHAPE), (dict(x=P + 8), ALIGN), (dict(ldx=258), ALIGN), (dict(r=P + 4), ALIGN), (dict(ldh=257), ALIGN),
    (dict(q=P + 4), ALIGN), (dict(ldq=260), ALIGN)])
def test_norm_refusals(lib, kw, code):
    a = dict(x=P, xdt=F32, ldx=256, r=P, rdt=F32, ldr=256, w=P, eps=1e-6, m=2, k=256, h=P, ldh=256, q=P, ldq=256, sx=P)
    a.update(kw)
    assert lib.tlx_add_rms_norm_q8(a["x"], a["xdt"], a["ldx"], a["r"], a["rdt"], a["ldr"], a["w"], a["eps"], a["m"],
                                   a["k"], a["h"], a["ldh"], a["q"], a["ldq"], a["sx"], None, None) == code


def test_front_end_needs_a_device():
    import torch

    from thunderllamax_b200 import paged
    if torch.cuda.is_available():
        pytest.skip("checks the machine without a GPU")
    for make in (lambda: paged.PagedAttention(4, 2, 128), lambda: paged.PageTable(2, 4, 8, 16)):
        with pytest.raises(_lib.TLXError):
            make()
    with pytest.raises(_lib.TLXError):
        paged.PagedCache(torch.zeros(2, 2, 16, 128), torch.zeros(2, 2, 16, 128))
