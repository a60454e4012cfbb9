"""Residual add + RMS norm + int8 tokens (tlx_add_rms_norm_q8) against 64 bits.

h is one fp32 addition rounded once.  y = h rstd w differs from 64 bits by a few fp32
roundings, below 2^-20 relative (the sum of up to 32768 squares is a tree of at most 4
sequential sums of 32 products per thread, then shuffles).  So the scales agree within
2^-19, and a code can differ by one only where y / s lies within 127 * 2^-18 of a
half-integer."""
import pytest
import torch

from thunderllamax_b200 import _lib, ops, prefill

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.require_device()


def reference(x, r, w, eps):
    h = x.double() + (r.double() if r is not None else 0.0)
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
    c = y.view(y.shape[0], -1, 128)
    s = c.abs().amax(-1).clamp(min=1e-6) / 127.0
    return h, c / s[..., None], s


def check(x, r, w, eps=1e-6, **kw):
    h_dtype = x.dtype if r is None else r.dtype
    rs = torch.empty((x.shape[0], x.shape[1] // 128), dtype=torch.int32, device="cuda")
    want_h = (x.float() + (r.float() if r is not None else 0.0)).to(h_dtype)
    ref_h, ref_q, ref_s = reference(x, r, w, eps)
    h, xq, sx = prefill.add_rms_norm_q8(x, r, w, eps, rs=rs, **kw)
    torch.cuda.synchronize()
    assert torch.equal(h, want_h)
    assert ((sx.double() - ref_s).abs() <= ref_s * 2.0 ** -19).all()
    q = xq.double().view_as(ref_q)
    assert (q.abs() <= 127).all()
    assert ((q - ref_q).abs() <= 0.5 + 127 * 2.0 ** -18).all()
    assert torch.equal(rs, xq.view(*rs.shape, 128).int().sum(-1, dtype=torch.int32))
    return h, xq, sx


@pytest.mark.parametrize("m,k", [(1, 128), (1, 5120), (2, 384), (11, 5120), (17, 2048), (300, 896), (5, 8192), (3, 8320),
                                 (2, 16512), (1, 32768)])
@pytest.mark.parametrize("xt,rt", [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F16, F32), (BF16, F32)])
def test_norm(m, k, xt, rt):
    g = torch.Generator(device="cuda").manual_seed(m * k)
    x = torch.randn((m, k), generator=g, device="cuda").to(xt)
    r = (2 * torch.randn((m, k), generator=g, device="cuda")).to(rt)
    w = 1 + 0.2 * torch.randn(k, generator=g, device="cuda")
    check(x, r, w)


def test_norm_strides_in_place_and_no_residual():
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn((40, 3, 640), generator=g, device="cuda")
    w = torch.rand(640, generator=g, device="cuda")
    check(wide[:, 1], wide[:, 2].contiguous(), w)
    check(wide[:, 0], None, w)
    r = torch.randn((40, 640), generator=g, device="cuda")
    want, _, _ = check(wide[:, 0], r, w)
    h, _, _ = prefill.add_rms_norm_q8(wide[:, 0], r, w, out=r)
    assert h.data_ptr() == r.data_ptr() and torch.equal(r, want)


def test_norm_matches_the_token_quantiser():
    # rows already normed to fp16 values: the same codes as act_quant_q8 gives for them
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((64, 1024), generator=g, device="cuda").half()
    ss = (x.float() ** 2).mean(-1, keepdim=True)
    one = torch.ones(1024, device="cuda")
    _, xq, sx = check(x, None, one, eps=0.0)
    y = (x.float() * torch.rsqrt(ss)).half()
    xq2, sx2, _ = prefill.act_quant_q8(y)
    assert ((xq.int() - xq2.int()).abs() <= 1).all() and torch.allclose(sx, sx2, rtol=2e-3)


def test_norm_zero_small_and_bad_rows():
    w = torch.ones(256, device="cuda")
    x = torch.zeros((5, 256), device="cuda")
    x[1, 3] = 1e-20
    x[2, 130] = float("nan")
    x[3, 1] = float("inf")
    x[4] = 3.0
    h, xq, sx = prefill.add_rms_norm_q8(x, None, w)
    torch.cuda.synchronize()
    assert (xq[:2] == 0).all() and (sx[:2] == torch.tensor(1e-6, device="cuda") * (1 / 127)).all()
    # a NaN shows in its whole row; an infinity makes the formula's factor 0, so it shows in its chunk
    assert sx[2].isnan().all() and sx[3, 0].isnan()
    assert (xq[4] == 127).all() and sx[4].isfinite().all()       # and in no other


def test_norm_feeds_the_w4a8_tier():
    from thunderllamax_b200.verify import synth_tiled
    m, k, n = 70, 512, 256
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn((m, k), generator=g, device="cuda") for _ in range(2))
    _, xq, sx = prefill.add_rms_norm_q8(x, r, torch.ones(k, device="cuda"))
    wg, wu = synth_tiled("iq3_xxs", n, k, 1), synth_tiled("iq3_xxs", n, k, 2)
    act = prefill.w4a8_gate_up(wg, wu, xq, sx, n, prefill.PrefillWorkspace(m, k))
    assert act.isfinite().all() and act.abs().max() > 0


def test_norm_refusals():
    x = torch.zeros((4, 256), device="cuda")
    w = torch.ones(256, device="cuda")
    bad = [dict(x=x[:, :200], residual=None, weight=w[:200]), dict(x=x.long(), residual=None, weight=w),
           dict(x=x, residual=x[:3], weight=w), dict(x=x, residual=None, weight=w.half()),
           dict(x=x, residual=None, weight=w, out=torch.zeros((4, 256), device="cuda", dtype=F16)),
           dict(x=x, residual=None, weight=w, eps=-1.0),
           dict(x=torch.zeros((4, 260), device="cuda")[:, 1:257], residual=None, weight=w),
           dict(x=torch.zeros((1, 33024), device="cuda"), residual=None, weight=torch.ones(33024, device="cuda")),
           dict(x=x, residual=None, weight=w, xq=torch.zeros((4, 256), dtype=torch.uint8, device="cuda")),
           dict(x=x, residual=None, weight=w, sx=torch.zeros((4, 3), device="cuda"))]
    for kw in bad:
        with pytest.raises(_lib.TLXError):
            prefill.add_rms_norm_q8(**kw)
