"""The operators as a transformer block uses them: norm -> router logits ->
softmax routing -> experts, and the dense 4-bit projections beside them."""
import numpy as np
import pytest
import torch

import moe_b200
import moe_oracle as mo
from moe_b200 import workloads
from test_gpu_routed import close, layer, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1, 40, 333])
def test_block(cuda_device, t):
    e, k, h = 24, 4, 512
    shape = workloads.MoeShape(t=t, hidden=h, inter=256, e_global=e, e_local=e)
    inp = workloads.make_inputs(shape, seed=t, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(t + 1)
    x = torch.randn(t, h, generator=g, device="cuda").to(torch.bfloat16)
    residual = torch.randn(t, h, generator=g, device="cuda").to(torch.bfloat16)
    gate = (0.05 * torch.randn(e, h, generator=g, device="cuda")).to(torch.bfloat16)
    norm_w = torch.ones(h, device="cuda", dtype=torch.bfloat16)
    up = (0.05 * torch.randn(256, h, generator=g, device="cuda")).to(torch.bfloat16)
    w4, s4 = moe_b200.quantize_fp4(up, "mxfp4")

    def block():
        q, s, y, res = moe_b200.rms_norm_quantize_1x128(x, norm_w, residual=residual, normed=True)
        idx, w = moe_b200.route_topk(moe_b200.router_logits(y, gate), k)
        out = torch.empty(t, h, dtype=torch.bfloat16, device="cuda")
        inp["hidden_states"], inp["hidden_states_scale"] = q, s
        moe_b200.run_routed(idx, w, *layer(inp), out, workspace=ws, deterministic=True)
        return q, s, y, res, idx, w, out, moe_b200.linear_fp4(y, w4, s4, "mxfp4")

    ws = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    q, s, y, res, idx, w, out, dense = block()
    torch.cuda.synchronize()
    # each step from the values it was given
    hid = x.double() + residual.double()
    exact = hid / (hid.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    assert ((y.double() - exact).abs() <= exact.abs() * (2.0 ** -8 + 2.0 ** -17)).all()
    p = torch.softmax(y.double() @ gate.double().t(), -1)
    # the logits' fp32 rounding may swap scores that close: compare the chosen scores
    top = p.sort(-1, descending=True)[0][:, :k]
    chosen = p.gather(1, idx.long())
    assert ((chosen - top).abs() <= top * 2.0 ** -12).all()
    assert ((w.double() - chosen / chosen.sum(-1, keepdim=True)).abs() <= 2.0 ** -12).all()
    close(out, oracle(inp, idx, w, e))
    va = moe_b200.dequantize_fp4(*moe_b200.quantize_fp4(y, "mxfp4"), "mxfp4", dtype=torch.float32).double()
    vb = moe_b200.dequantize_fp4(w4, s4, "mxfp4", dtype=torch.float32).double()
    ref, size = va @ vb.t(), va.abs() @ vb.abs().t()
    assert ((dense.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + size * 2.0 ** -15).all()
    # and the whole run captured: the same bits
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, (q, s, y, res, idx, w, out, dense)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
