"""Residual addition + RMS norm + FP8 1x128 output (``rms_norm_quantize_1x128``)
against the formula in 64 bits.

Bounds.  The kernel adds in fp32 (half an ulp, 2^-24 of h), sums the squares in
trees of less than 74 levels (each rounding 2^-24 of a sum of positive terms,
halved by the square root), and multiplies three times: y is within
(1 + 74 / 2 + 4) * 2^-24 < 2^-18 of its value.  Stored values add
half a step of their type (relative ``finfo.eps / 2``; absolute half of the
smallest subnormal below the normal range), the scale two roundings.
"""
import pytest
import torch

import moe_b200
from moe_b200 import workloads

pytestmark = pytest.mark.gpu
E = 2.0 ** -18


def half_step(v, dtype):
    f = torch.finfo(dtype)
    tiny = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150,
            torch.float8_e4m3fn: 2.0 ** -10}[dtype]
    return (v.abs() * (f.eps / 2)).clamp(min=tiny)


def reference(x, w, eps, residual):
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def check(x, w, eps, residual, q, scale, normed, res_out):
    h, y = reference(x, w, eps, residual)
    t, n = y.shape
    if residual is not None:
        assert res_out.dtype == residual.dtype
        assert ((res_out.double() - h).abs() <= half_step(h, residual.dtype) + h.abs() * 2 ** -24).all()
    if normed is not None:
        assert normed.dtype == x.dtype
        assert ((normed.double() - y).abs() <= half_step(y, x.dtype) * (1 + E) + y.abs() * E).all()
    s = (y.view(t, -1, 128).abs().amax(-1) / 448).clamp(min=1e-12).t()
    assert scale.shape == s.shape and ((scale.double() - s).abs() <= s * (E + 2 ** -23)).all()
    v = (y.view(t, -1, 128) / scale.double().t()[..., None]).view(t, n)
    assert ((q.double() - v).abs() <= half_step(v, torch.float8_e4m3fn) * (1 + E) + v.abs() * 2 * E).all()


def make(t, h, x, res, w, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    a = torch.randn(t, h, generator=g, device="cuda").to(x)
    r = None if res is None else (2 * torch.randn(t, h, generator=g, device="cuda")).to(res)
    return a, r, (1 + 0.1 * torch.randn(h, generator=g, device="cuda")).to(w)


B, F, S = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("x,res,w", [(B, None, B), (B, B, B), (B, S, S), (F, F, S), (F, S, F), (F, None, S)])
@pytest.mark.parametrize("t,h", [(1, 128), (1, 7168), (3, 384), (300, 512), (297, 2048), (901, 7168),
                                 (2, 65536), (400, 16384)])
def test_matches_the_formula(cuda_device, t, h, x, res, w):
    a, r, wt = make(t, h, x, res, w, 7 * t + h)
    check(a, wt, 1e-6, r, *moe_b200.rms_norm_quantize_1x128(a, wt, 1e-6, residual=r, normed=True))


def test_strided_rows_and_given_outputs(cuda_device):
    a, r, w = make(37, 512, B, B, B, 1)
    wide = torch.randn(37, 1536, device="cuda").to(B)
    x = wide[:, 512:1024]
    res = torch.randn(37, 640, device="cuda").to(B)[:, 128:]
    out = torch.full((37, 1024), 5.0, device="cuda", dtype=B)
    q, s, n, ro = moe_b200.rms_norm_quantize_1x128(x, w, 1e-5, residual=res, normed=out[:, 512:])
    check(x, w, 1e-5, res, q, s, n, ro)
    assert n.data_ptr() == out[:, 512:].data_ptr() and (out[:, :512] == 5).all()
    odd = torch.randn(37, 515, device="cuda").to(B)[:, 3:]     # rows off 16 bytes are copied
    check(odd, w, 1e-5, None, *moe_b200.rms_norm_quantize_1x128(odd, w, 1e-5, normed=True))
    t = torch.randn(512, 37, device="cuda").to(B).t()          # column-major input
    check(t, w, 1e-5, None, *moe_b200.rms_norm_quantize_1x128(t, w, 1e-5, normed=True))


def test_residual_and_input_in_place(cuda_device):
    a, r, w = make(65, 1024, B, S, B, 2)
    want = moe_b200.rms_norm_quantize_1x128(a, w, residual=r, normed=True)
    a2, r2 = a.clone(), r.clone()
    got = moe_b200.rms_norm_quantize_1x128(a2, w, residual=r2, residual_out=r2, normed=a2)
    assert got[2] is a2 and got[3] is r2
    for g, v in zip(got, want):
        assert torch.equal(g.view(torch.uint8), v.view(torch.uint8))


def test_quantised_as_the_layer_quantises(cuda_device):
    """With a power-of-two norm nothing rounds before the quantiser: the codes
    and scales are quantize_1x128's of the normed rows."""
    sign = torch.where(torch.rand(64, 512, device="cuda") < 0.5, -1.0, 1.0)
    w = torch.exp2(torch.randint(-6, 6, (512,), device="cuda").float()).to(B)
    q, s, n, _ = moe_b200.rms_norm_quantize_1x128((4 * sign).to(B), w, 0.0, normed=True)
    q2, s2 = moe_b200.quantize_1x128(n)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    q3, s3 = workloads.quantize_act_1x128(n)
    assert torch.equal(q.view(torch.uint8), q3.view(torch.uint8)) and torch.equal(s, s3)


def test_zero_and_non_finite_rows(cuda_device):
    a, r, w = make(8, 512, B, B, B, 3)
    a[1], r[1] = 0, 0
    a[2, 5] = float("nan")
    a[3, 130] = float("inf")
    q, s, n, ro = moe_b200.rms_norm_quantize_1x128(a, w, residual=r, normed=True)
    assert (n[1] == 0).all() and (q[1].float() == 0).all() and (s[:, 1] == torch.tensor(1e-12)).all()
    assert n[2].isnan().all() and s[:, 2].isnan().all() and q[2].float().isnan().all()
    # rsqrt(inf) = 0: the infinity's own value is NaN, the others 0
    assert n[3, 130].isnan() and n[3].isnan().sum() == 1 and s[1, 3].isnan()
    assert (s[[0, 2, 3], 3] == torch.tensor(1e-12)).all()
    ok = [0, 4, 5, 6, 7]
    check(a[ok], w, 1e-6, r[ok], q[ok], s[:, ok], n[ok], ro[ok])


def test_empty_batch_stream_and_graph(cuda_device):
    w = torch.ones(256, device="cuda", dtype=B)
    q, s, n, ro = moe_b200.rms_norm_quantize_1x128(torch.empty(0, 256, device="cuda", dtype=B), w, normed=True)
    assert q.shape == (0, 256) and s.shape == (2, 0) and n.shape == (0, 256) and ro is None
    a, r, w = make(50, 1024, F, F, F, 4)
    want = moe_b200.rms_norm_quantize_1x128(a, w, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = moe_b200.rms_norm_quantize_1x128(a, w, residual=r)
    side.synchronize()
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and got[2] is None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = moe_b200.rms_norm_quantize_1x128(a, w, residual=r)
    a2, r2, _ = make(50, 1024, F, F, F, 5)
    a.copy_(a2), r.copy_(r2)
    graph.replay()
    torch.cuda.synchronize()
    check(a2, w, 1e-6, r2, got[0], got[1], None, got[3])


def test_offsets_past_32_bits(cuda_device):
    h, t = 7168, 2 ** 31 // 7168 + 100
    x = torch.ones(t, h, device="cuda", dtype=B)
    x[-200:] = make(200, h, B, None, B, 6)[0]
    w = torch.ones(h, device="cuda", dtype=B)
    q, s, n, _ = moe_b200.rms_norm_quantize_1x128(x, w, normed=True)
    check(x[-200:], w, 1e-6, None, q[-200:], s[:, -200:], n[-200:], None)
    assert (n[:-200] == 1).all()


@pytest.mark.parametrize("t,h", [(5, 256), (700, 2048), (700, 7168)])
@pytest.mark.parametrize("at,pad", [(0, 0), (4, 4), (4, 0), (0, 4), (8, 8)])
def test_fp32_rows_of_any_alignment(cuda_device, t, h, at, pad):
    """fp32 weight and residual 16 or 32 bytes aligned, rows of either stride, in place
    and not: the same bits, and nothing written beside the rows."""
    g = torch.Generator(device="cuda").manual_seed(t + h)
    x = torch.randn(t, h, generator=g, device="cuda").bfloat16()
    res, w = torch.randn(t, h, generator=g, device="cuda"), torch.rand(h, generator=g, device="cuda")
    want = moe_b200.rms_norm_quantize_1x128(x, w, residual=res, normed=True)
    wide = torch.full((t, at + h + pad), 9.0, device="cuda")
    wide[:, at:at + h] = res
    wb = torch.full((at + h,), 9.0, device="cuda")
    wb[at:] = w
    out = torch.full_like(wide, 9.0)
    got = moe_b200.rms_norm_quantize_1x128(x, wb[at:], residual=wide[:, at:at + h], residual_out=out[:, at:at + h], normed=True)
    again = moe_b200.rms_norm_quantize_1x128(x, wb[at:], residual=wide[:, at:at + h], residual_out=wide[:, at:at + h],
                                             normed=True)
    for a in (got, again):
        for v, e in zip(a, want):
            assert torch.equal(v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v,
                               e.view(torch.uint8) if e.dtype == torch.float8_e4m3fn else e)
    for b in (wide, out):
        assert (b[:, :at] == 9).all() and (b[:, at + h:] == 9).all()
