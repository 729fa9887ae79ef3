"""The Python side of the operators around the layer, on the CPU."""
import ctypes

import pytest
import torch

from moe_b200 import _lib, ops


LIBRARY = _lib.load()


def size(fmt, t, k):
    n = ctypes.c_size_t()
    assert LIBRARY.moe_fp4_linear_workspace_size(fmt, t, k, ctypes.byref(n)) == 0
    return n.value


class Library:
    """The library, but products want `more` bytes of workspace."""

    def __init__(self, more):
        self.more = more

    def moe_fp4_linear_workspace_size(self, fmt, t, k, n):
        n._obj.value = size(fmt, t, k) + self.more
        return 0


@pytest.mark.parametrize("more", [0, 768])
@pytest.mark.parametrize("t", [1, 4, 5, 16, 129])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_the_library_tells_the_workspace_size(monkeypatch, fmt, t, more):
    """How much a product wants, and from how many tokens on, is the library's to say."""
    k, n = 96, 8
    want = size(ops._FORMATS[fmt], t, k) + more
    monkeypatch.setattr(ops, "_gpu", lambda t, name: 0)
    monkeypatch.setattr(ops, "_same", lambda t, name, index: None)
    got = []
    monkeypatch.setattr(ops, "_call", lambda name, index, *args: got.append((name, args)))
    if more:
        monkeypatch.setattr(_lib, "load", lambda: Library(more))
    cached = getattr(ops, "_linear_workspace", None)
    if cached is not None:
        cached.cache_clear()
    try:
        ops.linear_fp4(torch.zeros(t, k, dtype=torch.bfloat16), torch.zeros(n, k // 2, dtype=torch.uint8),
                       torch.zeros(ops.fp4_scales_shape(n, k, fmt), dtype=torch.uint8), fmt)
    finally:
        if cached is not None:
            cached.cache_clear()
    (name, args), = got
    assert name == "moe_fp4_linear" and args[-1] == want and (args[-2] is None) == (want == 0)


BF = torch.zeros(4, 256, dtype=torch.bfloat16)
W = torch.ones(256, dtype=torch.bfloat16)
CODES, SCALES = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)


@pytest.mark.parametrize("call,message", [
    (lambda: ops.rms_norm_quantize_1x128(BF, W), "x must be a CUDA tensor"),
    (lambda: ops.rms_norm_quantize_1x128(BF.float(), W), "x must be a bf16 or fp16"),
    (lambda: ops.rms_norm_quantize_1x128(BF[0], W), "x must be a bf16 or fp16"),
    (lambda: ops.rms_norm_quantize_1x128(BF[:, :100], W[:100]), "H must be a multiple of 128"),
    (lambda: ops.rms_norm_quantize_1x128(BF[:, :0], W[:0]), "H must be a multiple of 128"),
    (lambda: ops.rms_norm_quantize_1x128(BF, W[:128]), "weight must be"),
    (lambda: ops.rms_norm_quantize_1x128(BF, W.half()), "weight must be"),
    (lambda: ops.rms_norm_quantize_1x128(BF, W, residual_out=BF), "residual_out needs a residual"),
    (lambda: ops.route_topk(BF, 4), "logits must be a CUDA tensor"),
    (lambda: ops.route_topk(BF[0], 4), "logits must be fp32, bf16 or fp16"),
    (lambda: ops.route_topk(BF.int(), 4), "logits must be fp32, bf16 or fp16"),
    (lambda: ops.route_topk(BF, 4, score="tanh"), "score must be"),
    (lambda: ops.route_topk(BF, 4, group_score="mean"), "group_score must be"),
    (lambda: ops.route_topk(BF, 0), "top_k must be 1 to 32"),
    (lambda: ops.route_topk(BF, 33), "top_k must be 1 to 32"),
    (lambda: ops.quantize_fp4(BF), "x must be a CUDA tensor"),
    (lambda: ops.quantize_fp4(BF, "fp4"), "fmt must be"),
    (lambda: ops.quantize_fp4(BF[:, :48]), "K must be a multiple of 32"),
    (lambda: ops.quantize_fp4(BF.double()), "x must be fp32, bf16 or fp16"),
    (lambda: ops.quantize_fp4(BF[0]), "x must be fp32, bf16 or fp16"),
    (lambda: ops.dequantize_fp4(CODES, SCALES), "input_codes must be a CUDA tensor"),
    (lambda: ops.dequantize_fp4(CODES, SCALES, "nf4"), "fmt must be"),
    (lambda: ops.dequantize_fp4(CODES.int(), SCALES), "input_codes must be uint8"),
    (lambda: ops.dequantize_fp4(CODES[0], SCALES), "input_codes must be uint8"),
    (lambda: ops.dequantize_fp4(CODES[:, :8], SCALES), "K must be a multiple of 32"),
    (lambda: ops.dequantize_fp4(CODES, SCALES[0]), "input_scales must be uint8"),
    (lambda: ops.dequantize_fp4(CODES, SCALES.int()), "input_scales must be uint8"),
    (lambda: ops.dequantize_fp4(CODES, SCALES.repeat_interleave(2, -1)[..., ::2]), "contiguous and 16-byte aligned"),
    (lambda: ops.dequantize_fp4(CODES, torch.zeros(520, dtype=torch.uint8)[8:].view(SCALES.shape)),
     "contiguous and 16-byte aligned"),
    (lambda: ops.matmul_fp4(CODES, SCALES, CODES, SCALES), "a_codes must be a CUDA tensor"),
    (lambda: ops.matmul_fp4(CODES, SCALES, CODES, SCALES, "int4"), "fmt must be"),
    (lambda: ops.linear_fp4(BF, CODES, SCALES), "w_codes must be a CUDA tensor"),
    (lambda: ops.linear_fp4(BF, CODES, SCALES, "mxfp8"), "fmt must be"),
    (lambda: ops.fp4_scales_shape(4, 64, "fp8"), "fmt must be"),
])
def test_refusals_name_what_is_wrong(call, message):
    with pytest.raises(AssertionError, match=message):
        call()
