"""Arguments that the operators around the layer refuse, on the CPU: the C ABI's
status codes before any CUDA call, and the Python layer's AssertionErrors."""
import ctypes

import pytest
import torch

import moe_b200
from moe_b200 import _lib

SHAPE, ARG, ALIGN, WS = _lib.MOE_ERR_SHAPE, _lib.MOE_ERR_INVALID_ARG, _lib.MOE_ERR_ALIGNMENT, _lib.MOE_ERR_WORKSPACE
P = 1 << 20      # a 16-byte aligned address that no refused call reads


def norm(**kw):
    d = dict(x=P, xd=1, ldx=512, r=None, rd=1, ldr=512, w=P, wd=1, eps=1e-6, t=4, h=512, ro=None, ldro=512, n=None,
             ldn=512, q=P, s=P, stream=None)
    d.update(kw)
    return _lib.load().moe_rms_norm_1x128(*d.values())


@pytest.mark.parametrize("bad,want", [
    (dict(t=-1), SHAPE), (dict(h=0), SHAPE), (dict(h=100), SHAPE), (dict(h=65664), SHAPE), (dict(t=(1 << 24) + 1), SHAPE),
    (dict(xd=0), ARG), (dict(xd=7), ARG), (dict(wd=2), ARG), (dict(r=P, ro=P, rd=2), ARG), (dict(r=P), ARG), (dict(ro=P), ARG),
    (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(x=None), ARG), (dict(w=None), ARG), (dict(q=None), ARG),
    (dict(s=None), ARG), (dict(ldx=511), SHAPE), (dict(ldx=516), SHAPE), (dict(n=P, ldn=500), SHAPE),
    (dict(r=P, ro=P, ldr=516), SHAPE), (dict(r=P, ro=P, rd=0, ldr=516, ldro=518), SHAPE), (dict(x=P + 8), ALIGN),
    (dict(q=P + 8), ALIGN), (dict(s=P + 2), ALIGN), (dict(n=P + 2), ALIGN)])
def test_norm(bad, want):
    assert norm(**bad) == want


def topk(**kw):
    d = dict(x=P, dt=0, ld=64, b=None, bd=0, t=4, e=64, k=8, score=0, ng=1, tg=1, gs=0, renorm=1, f=1.0, i=P, w=P,
             stream=None)
    d.update(kw)
    return _lib.load().moe_route_topk(*d.values())


@pytest.mark.parametrize("bad,want", [
    (dict(t=-1), SHAPE), (dict(t=(1 << 24) + 1), SHAPE), (dict(e=0), SHAPE), (dict(e=1025, ld=1025), SHAPE), (dict(k=0), SHAPE),
    (dict(k=33), SHAPE), (dict(e=4, k=5), SHAPE), (dict(ng=0), SHAPE), (dict(ng=3), SHAPE), (dict(ng=64, tg=64), SHAPE),
    (dict(ng=8, tg=9), SHAPE), (dict(ng=8, tg=0), SHAPE), (dict(ng=16, tg=1), SHAPE), (dict(ld=63), SHAPE),
    (dict(e=32, ng=32, tg=16), SHAPE), (dict(dt=3), ARG), (dict(b=P, bd=4), ARG), (dict(score=2), ARG), (dict(gs=2), ARG),
    (dict(x=None), ARG), (dict(i=None), ARG), (dict(w=None), ARG), (dict(x=P + 2), ALIGN), (dict(x=P + 1, dt=1), ALIGN),
    (dict(b=P + 2), ALIGN), (dict(i=P + 1), ALIGN), (dict(w=P + 2), ALIGN)])
def test_topk(bad, want):
    assert topk(**bad) == want


def quant(**kw):
    d = dict(x=P, dt=1, ld=64, r=4, k=64, fmt=1, g=None, c=P, s=P, stream=None)
    d.update(kw)
    return _lib.load().moe_fp4_quantize(*d.values())


@pytest.mark.parametrize("bad,want", [
    (dict(r=-1), SHAPE), (dict(r=(1 << 24) + 1), SHAPE), (dict(k=0), SHAPE), (dict(k=48), SHAPE), (dict(k=65568, ld=65568), SHAPE),
    (dict(ld=56), SHAPE), (dict(ld=68), SHAPE), (dict(dt=0, ld=66), SHAPE), (dict(fmt=2), ARG), (dict(dt=3), ARG),
    (dict(fmt=0, g=P), ARG), (dict(x=None), ARG), (dict(c=None), ARG), (dict(s=None), ARG), (dict(x=P + 2), ALIGN),
    (dict(c=P + 8), ALIGN), (dict(s=P + 8), ALIGN), (dict(g=P + 2), ALIGN)])
def test_quantize(bad, want):
    assert quant(**bad) == want


def dequant(**kw):
    d = dict(c=P, ld=32, s=P, r=4, k=64, fmt=1, g=None, o=P, dt=1, stream=None)
    d.update(kw)
    return _lib.load().moe_fp4_dequantize(*d.values())


@pytest.mark.parametrize("bad,want", [
    (dict(k=16), SHAPE), (dict(ld=16), SHAPE), (dict(ld=40), SHAPE), (dict(fmt=-1), ARG), (dict(dt=9), ARG),
    (dict(fmt=0, g=P), ARG), (dict(c=None), ARG), (dict(o=None), ARG), (dict(o=P + 8), ALIGN), (dict(c=P + 4), ALIGN)])
def test_dequantize(bad, want):
    assert dequant(**bad) == want


def matmul(**kw):
    d = dict(a=P, lda=32, sa=P, ga=None, b=P, ldb=32, sb=P, gb=None, fmt=1, t=4, n=8, k=64, o=P, dt=1, ldo=8, stream=None)
    d.update(kw)
    return _lib.load().moe_fp4_matmul(*d.values())


def linear(**kw):
    d = dict(x=P, xd=1, ldx=64, gx=None, b=P, ldb=32, sb=P, gb=None, fmt=1, t=4, n=8, k=64, o=P, dt=1, ldo=8, ws=P,
             wb=1 << 16, stream=None)
    d.update(kw)
    return _lib.load().moe_fp4_linear(*d.values())


@pytest.mark.parametrize("bad,want", [
    (dict(t=-1), SHAPE), (dict(t=(1 << 22) + 1), SHAPE), (dict(n=0), SHAPE), (dict(k=40), SHAPE), (dict(ldb=16), SHAPE),
    (dict(ldb=40), SHAPE), (dict(ldo=7), SHAPE), (dict(fmt=5), ARG), (dict(dt=5), ARG), (dict(fmt=0, gb=P), ARG),
    (dict(b=None), ARG), (dict(sb=None), ARG), (dict(o=None), ARG), (dict(b=P + 8), ALIGN), (dict(sb=P + 8), ALIGN),
    (dict(gb=P + 1), ALIGN), (dict(o=P + 1), ALIGN), (dict(dt=0, o=P + 2), ALIGN)])
def test_products(bad, want):
    assert matmul(**bad) == want
    assert linear(**bad) == want


def test_more_product_refusals():
    assert matmul(lda=16) == SHAPE and matmul(lda=40) == SHAPE
    assert matmul(a=None) == ARG and matmul(sa=None) == ARG and matmul(fmt=0, ga=P) == ARG
    assert matmul(a=P + 8) == ALIGN and matmul(sa=P + 8) == ALIGN and matmul(ga=P + 2) == ALIGN
    assert linear(t=16, ws=None) == WS and linear(t=16, wb=100) == WS and linear(t=16, ws=P + 128) == ALIGN
    assert linear(x=None) == ARG and linear(xd=4) == ARG and linear(ldx=60) == SHAPE and linear(x=P + 2) == ALIGN
    n = ctypes.c_size_t()
    assert _lib.load().moe_fp4_scales_size(1, 129, 80 + 16, ctypes.byref(n)) == 0 and n.value == 2 * 2 * 512
    assert _lib.load().moe_fp4_scales_size(0, 129, 96, ctypes.byref(n)) == 0 and n.value == 2 * 512
    assert _lib.load().moe_fp4_scales_size(0, 129, 95, ctypes.byref(n)) == SHAPE
    assert _lib.load().moe_fp4_linear_workspace_size(1, 16, 64, ctypes.byref(n)) == 0 and n.value == 512 + 512
    assert _lib.load().moe_fp4_linear_workspace_size(1, 3, 64, ctypes.byref(n)) == 0 and n.value == 0


@pytest.mark.parametrize("x,ldx,t,o,ldo,dt", [
    (P, 64, 4, P, 64, 1), (P, 64, 1, P + 112, 64, 1), (P + 112, 64, 1, P, 64, 1), (P, 64, 40, P + 39 * 128, 64, 1),
    (P, 128, 4, P + 112, 128, 1), (P + 128, 128, 4, P + 256 - 16, 128, 1), (P, 128, 4, P + 240, 64, 0),
    (P, 128, 4, P + 128, 64, 1), (P + 16, 64, 2, P + 128, 60, 1)])
def test_product_into_its_own_input(x, ldx, t, o, ldo, dt):
    """Every block of a small product reads x while others store: out inside x's rows."""
    assert linear(x=x, ldx=ldx, t=t, o=o, ldo=ldo, n=60, dt=dt) == ARG


def test_empty_batches_need_no_gpu():
    assert norm(t=0) == 0 and topk(t=0) == 0 and quant(r=0) == 0 and dequant(r=0) == 0
    assert matmul(t=0) == 0 and linear(t=0) == 0


def test_routed_forward_refusals():
    a = _lib.MoeFwdArgs()
    for k, v in dict(T=4, H=512, I=256, E_global=60, E_local=60, top_k=8, n_group=0, topk_group=0).items():
        setattr(a, k, v)
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.moe_fp8_workspace_size(a, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.moe_fp8_forward_routed(None, None, None, None) == ARG
    assert lib.moe_fp8_forward_routed(a, P, P, None) == ARG            # no tensors
    assert lib.moe_fp8_forward(a, None) == SHAPE                       # needs the router's groups
    for k, v in dict(top_k=9, E_global=300, topk_group=1, local_expert_offset=1).items():
        old = getattr(a, k)
        setattr(a, k, v)
        assert lib.moe_fp8_forward_routed(a, P, P, None) == SHAPE, k
        setattr(a, k, old)
    a.T = 0
    assert lib.moe_fp8_forward_routed(a, None, None, None) == 0


def test_python_refusals():
    bf = torch.zeros(4, 256, dtype=torch.bfloat16)
    w = torch.ones(256, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    m = moe_b200
    calls = [
        lambda: m.rms_norm_quantize_1x128(bf, w), lambda: m.rms_norm_quantize_1x128(bf.float(), w),
        lambda: m.rms_norm_quantize_1x128(bf[0], w), lambda: m.rms_norm_quantize_1x128(bf[:, :100], w[:100]),
        lambda: m.rms_norm_quantize_1x128(bf, w[:128]), lambda: m.rms_norm_quantize_1x128(bf, w.half()),
        lambda: m.rms_norm_quantize_1x128(bf, w, residual_out=bf),
        lambda: m.route_topk(bf, 4), lambda: m.route_topk(bf[0], 4), lambda: m.route_topk(bf.int(), 4),
        lambda: m.route_topk(bf, 4, score="tanh"), lambda: m.route_topk(bf, 4, group_score="mean"),
        lambda: m.quantize_fp4(bf), lambda: m.quantize_fp4(bf, "fp4"), lambda: m.quantize_fp4(bf[:, :48]),
        lambda: m.quantize_fp4(bf.double()), lambda: m.quantize_fp4(bf, "mxfp4", global_scale=torch.ones(1)),
        lambda: m.quantize_fp4(bf, global_scale=torch.ones(2)), lambda: m.quantize_fp4(bf, global_scale=w[:1]),
        lambda: m.dequantize_fp4(codes, scales), lambda: m.dequantize_fp4(codes.int(), scales),
        lambda: m.dequantize_fp4(codes, scales[0]), lambda: m.dequantize_fp4(codes[:, :8], scales),
        lambda: m.dequantize_fp4(codes, scales, dtype=torch.float64),
        lambda: m.matmul_fp4(codes, scales, codes, scales), lambda: m.matmul_fp4(codes, scales, codes[:, :16], scales),
        lambda: m.linear_fp4(bf, codes, scales), lambda: m.linear_fp4(bf[:, :64], codes, scales, "mxfp8"),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was accepted")
