"""The operators around the layer give the same bits on every call and beside other work."""
import pytest
import torch

import moe_b200

pytestmark = pytest.mark.gpu


def bits(outputs):
    return [t.view(torch.uint8) for t in outputs if t is not None]


@pytest.mark.parametrize("t", [7, 3000])
def test_same_bits_every_time(cuda_device, t):
    gen = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(t, 2048, generator=gen, device="cuda").to(torch.bfloat16)
    res = torch.randn(t, 2048, generator=gen, device="cuda").to(torch.bfloat16)
    w = torch.rand(2048, generator=gen, device="cuda").to(torch.bfloat16)
    logits, bias = torch.randn(t, 512, generator=gen, device="cuda"), torch.rand(512, generator=gen, device="cuda")
    g = x.abs().max().float().reshape(1) / 2688
    calls = [lambda: moe_b200.rms_norm_quantize_1x128(x, w, residual=res, normed=True),
             lambda: moe_b200.route_topk(logits, 8, bias=bias, n_group=8, topk_group=4, score="sigmoid"),
             lambda: moe_b200.quantize_fp4(x, "nvfp4", global_scale=g), lambda: moe_b200.quantize_fp4(x, "mxfp4")]
    want = [bits(c()) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(10):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(bits(c()))
    torch.cuda.synchronize()
    for i, outputs in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(outputs, want[i % len(calls)]))
