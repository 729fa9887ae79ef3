"""Arguments on the GPU that the operators around the layer refuse, by what is wrong with
them; the same calls without the fault are accepted."""
import pytest
import torch

import moe_b200 as m

pytestmark = pytest.mark.gpu
B = torch.bfloat16


def zeros(*shape, dtype=B):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def refused(fn, message, **kw):
    with pytest.raises(AssertionError, match=message):
        fn(**kw)


def test_norm(cuda_device):
    x, w = zeros(4, 256), zeros(256)

    def call(x=x, w=w, eps=1e-6, **kw):
        return m.rms_norm_quantize_1x128(x, w, eps, **kw)

    call(residual=zeros(4, 256, dtype=torch.float32), normed=zeros(4, 256), scale=zeros(2, 4, dtype=torch.float32),
         q=zeros(4, 256, dtype=torch.float8_e4m3fn))
    refused(call, "weight must be on cuda:0", w=w.cpu())
    refused(call, "residual must be", residual=zeros(3, 256))
    refused(call, "residual must be", residual=zeros(4, 256, dtype=torch.float16))
    refused(call, "residual must be on cuda:0", residual=zeros(4, 256).cpu())
    refused(call, "residual_out must be", residual=x, residual_out=zeros(4, 256, dtype=torch.float32))
    refused(call, "residual_out must be on cuda:0", residual=x, residual_out=zeros(4, 256).cpu())
    refused(call, "residual_out must have contiguous, 16-byte aligned rows", residual=x, residual_out=zeros(4, 260)[:, 2:258])
    refused(call, "normed must be", normed=zeros(4, 128))
    refused(call, "normed must be", normed=zeros(4, 256, dtype=torch.float32))
    refused(call, "normed must have contiguous, 16-byte aligned rows", normed=zeros(256, 4).t())
    refused(call, "normed must have contiguous, 16-byte aligned rows", normed=zeros(1, 256).expand(4, 256))
    refused(call, "q must be", q=zeros(4, 256, dtype=torch.uint8))
    refused(call, "q must be contiguous", q=zeros(4, 512, dtype=torch.float8_e4m3fn)[:, :256])
    refused(call, "scale must be", scale=zeros(4, 2, dtype=torch.float32))
    refused(call, "scale must be contiguous", scale=zeros(4, 2, dtype=torch.float32).t())
    refused(call, "moe_rms_norm_1x128", eps=-1e-6)
    refused(call, "moe_rms_norm_1x128", eps=float("nan"))
    refused(call, "moe_rms_norm_1x128", x=zeros(1, 65664), w=zeros(65664))


def test_route(cuda_device):
    x = zeros(4, 64)

    def call(x=x, k=4, **kw):
        return m.route_topk(x, k, **kw)

    call(bias=zeros(64), topk_idx=zeros(4, 4, dtype=torch.int32), topk_weights=zeros(4, 4, dtype=torch.float32))
    refused(call, "bias must be", bias=zeros(63))
    refused(call, "bias must be", bias=zeros(64, dtype=torch.float64))
    refused(call, "bias must be on cuda:0", bias=zeros(64).cpu())
    refused(call, "topk_idx must be", topk_idx=zeros(4, 4, dtype=torch.int64))
    refused(call, "topk_idx must be contiguous", topk_idx=zeros(4, 4, dtype=torch.int32).t())
    refused(call, "topk_weights must be", topk_weights=zeros(4, 3, dtype=torch.float32))
    refused(call, "topk_weights must be on cuda:0", topk_weights=zeros(4, 4, dtype=torch.float32).cpu())
    for kw in (dict(n_group=3), dict(n_group=0), dict(n_group=8, topk_group=9), dict(n_group=8, topk_group=0),
               dict(n_group=64), dict(n_group=16, topk_group=1, k=5), dict(x=zeros(4, 1025)), dict(x=zeros(4, 3)),
               dict(x=zeros(4, 32), n_group=32, topk_group=16)):
        refused(call, "moe_route_topk", **kw)


def test_quantize_and_back(cuda_device):
    x = zeros(4, 64)

    def quantize(fmt="nvfp4", **kw):
        return m.quantize_fp4(x, fmt, **kw)

    codes, scales = quantize(global_scale=torch.ones(1, device="cuda"))
    refused(quantize, "global_scale belongs to nvfp4", fmt="mxfp4", global_scale=torch.ones(1, device="cuda"))
    refused(quantize, "global_scale must be one float32", global_scale=torch.ones(2, device="cuda"))
    refused(quantize, "global_scale must be one float32", global_scale=torch.ones(1, device="cuda", dtype=B))
    refused(quantize, "global_scale must be on cuda:0", global_scale=torch.ones(1))
    refused(quantize, "codes must be", codes=zeros(4, 64, dtype=torch.uint8))
    refused(quantize, "codes must be contiguous", codes=zeros(4, 64, dtype=torch.uint8)[:, :32])
    refused(quantize, "scales must be", scales=zeros(1, 512, dtype=torch.uint8))

    def back(fmt="nvfp4", scales=scales, **kw):
        return m.dequantize_fp4(codes, scales, fmt, **kw)

    back(out=zeros(4, 64))
    refused(back, "input_scales must be on cuda:0", scales=scales.cpu())
    refused(back, "dtype must be", dtype=torch.float64)
    refused(back, "out must be", out=zeros(4, 64, dtype=torch.float32))
    refused(back, "out must be contiguous", out=zeros(4, 128)[:, :64])
    refused(back, "global_scale belongs to nvfp4", fmt="mxfp4", global_scale=torch.ones(1, device="cuda"))


def test_products(cuda_device):
    x = zeros(4, 64)
    a, b = m.quantize_fp4(x), m.quantize_fp4(zeros(24, 64))
    other = m.quantize_fp4(zeros(24, 32))
    g = torch.ones(1, device="cuda")

    def matmul(a=a, b=b, fmt="nvfp4", **kw):
        return m.matmul_fp4(*a, *b, fmt, **kw)

    def linear(x=x, b=b, fmt="nvfp4", **kw):
        return m.linear_fp4(x, *b, fmt, **kw)

    matmul(out=zeros(4, 32)[:, 3:27], a_global_scale=g), linear(out=zeros(4, 24), w_global_scale=g)
    refused(matmul, "a and b must have the same K", b=other)
    refused(matmul, "b_codes must be a CUDA tensor", b=(b[0].cpu(), b[1].cpu()))
    mx = m.quantize_fp4(x, "mxfp4"), m.quantize_fp4(zeros(24, 64), "mxfp4")
    refused(matmul, "a_global_scale belongs to nvfp4", a=mx[0], b=mx[1], fmt="mxfp4", a_global_scale=g)
    refused(linear, "w_global_scale belongs to nvfp4", b=mx[1], fmt="mxfp4", w_global_scale=g)
    for fn in (matmul, linear):
        refused(fn, "dtype must be", dtype=torch.float64)
        refused(fn, "out must be", out=zeros(4, 25))
        refused(fn, "out must be", out=zeros(4, 24, dtype=torch.float16))
        refused(fn, "out must be on cuda:0", out=zeros(4, 24).cpu())
        refused(fn, "out must have contiguous rows", out=zeros(4, 48)[:, ::2])
        refused(fn, "rows of out must not overlap", out=zeros(1, 24).expand(4, 24))
    refused(linear, r"x must be \[T, 64\]", x=zeros(4, 96))
    refused(linear, "x must be fp32, bf16 or fp16", x=zeros(64))
    refused(linear, "x must be fp32, bf16 or fp16", x=zeros(4, 64, dtype=torch.float64))
    refused(linear, "x must be on cuda:0", x=x.cpu())
    refused(linear, "moe_fp4_linear", b=(zeros(0, 32, dtype=torch.uint8), zeros(0, 1, 32, 4, 4, dtype=torch.uint8)))
