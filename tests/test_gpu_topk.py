"""Routing to experts (``route_topk``) against its definition in 64 bits.

The chosen experts and their order must be equal.  Weights: expf is within two
ulps, the shift by the row's maximum rounds once (half an ulp of at most 32, the
spread of these logits), sums and quotients add a few roundings: less than
(4 + 32 + 8) * 2^-24 < 2^-18 relative.
"""
import math

import pytest
import torch

import moe_b200
from moe_b200 import workloads

pytestmark = pytest.mark.gpu


def reference(x, k, bias=None, score="softmax", n_group=1, topk_group=1, group_score="top2",
              renormalize=True, factor=1.0):
    x = x.double().cpu()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    t, e = x.shape
    if score == "sigmoid":
        s = torch.sigmoid(x)
    else:
        m = x.amax(-1, keepdim=True)
        s = torch.where(x == m, torch.ones_like(x), torch.exp(x - m))
        s = torch.where(m == -math.inf, torch.zeros_like(s), s)
        total = s.sum(-1, keepdim=True)
        s = s / torch.where(total > 0, total, torch.ones_like(total))
    # without a bias and without sums the order is the logits' own
    c = x if bias is None and not (topk_group < n_group and group_score == "top2") else \
        s if bias is None else s + bias.double().cpu()
    c = torch.where(c.isnan(), torch.full_like(c, -math.inf), c)
    open_ = torch.ones(t, e, dtype=torch.bool)
    if topk_group < n_group:
        per = c.view(t, n_group, -1)
        best = per.sort(-1, descending=True)[0]
        g = best[..., 0] if group_score == "max" else \
            torch.where(best[..., 0] == math.inf, best[..., 0], best[..., 0] + best[..., 1])
        keep = g.sort(dim=-1, descending=True, stable=True)[1][:, :topk_group]
        open_ = torch.zeros(t, n_group, dtype=torch.bool).scatter_(1, keep, True)
        open_ = open_[..., None].expand(t, n_group, e // n_group).reshape(t, e)
    idx = torch.empty(t, k, dtype=torch.int64)
    order = torch.arange(e)
    for r in range(t):   # open experts first, then by score, then by id
        ids = order[open_[r]]
        idx[r] = ids[c[r][ids].sort(descending=True, stable=True)[1][:k]]
    w = s.gather(1, idx)
    if renormalize:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return idx, w * factor


def run_and_check(x, k, factor=1.0, **kw):
    idx, w = moe_b200.route_topk(x, k, routed_scaling_factor=factor, **kw)
    ref_idx, ref_w = reference(x, k, factor=factor, **kw)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(idx.cpu().long(), ref_idx), (idx.cpu().long() != ref_idx).nonzero()[:4]
    assert ((w.double().cpu() - ref_w).abs() <= ref_w.abs() * 2 ** -18 + 1e-38).all()
    return idx, w


def logits(t, e, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(t, e, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k,n_group,topk_group,group_score", [
    (1, 1, 1, 1, 1, "max"), (1, 8, 2, 1, 1, "max"), (5, 32, 32, 1, 1, "max"), (33, 60, 4, 1, 1, "top2"),
    (64, 256, 8, 8, 4, "top2"), (64, 160, 6, 8, 3, "max"), (17, 257, 8, 1, 1, "max"), (9, 96, 5, 32, 7, "max"),
    (31, 72, 8, 3, 1, "top2"), (40, 512, 10, 16, 5, "top2"), (13, 1024, 32, 2, 1, "max"), (7, 1000, 3, 5, 2, "top2"),
])
def test_matches_the_definition(cuda_device, t, e, k, n_group, topk_group, group_score, score, dtype):
    x = logits(t, e, dtype, t + e)
    kw = dict(score=score, n_group=n_group, topk_group=topk_group, group_score=group_score)
    bias = 0.1 * torch.randn(e, device="cuda", generator=torch.Generator(device="cuda").manual_seed(e))
    for renorm in (True, False):
        run_and_check(x, k, renormalize=renorm, factor=2.5, **kw)
        run_and_check(x, k, renormalize=renorm, bias=bias, **kw)
    run_and_check(x, k, bias=bias.to(torch.bfloat16), **kw)
    run_and_check(x, k, bias=bias.half(), **kw)


def test_many_tokens(cuda_device):
    run_and_check(logits(9001, 128, torch.float32, 1), 8)
    run_and_check(logits(2777, 256, torch.float32, 2), 8, score="sigmoid", n_group=8, topk_group=4, factor=2.5,
                  bias=0.1 * torch.randn(256, device="cuda"))


def test_ties_go_to_the_lowest_id(cuda_device):
    x = torch.zeros(3, 200, device="cuda")
    x[1, 150:] = 1.0
    x[2, ::3] = -1.0
    for kw in (dict(), dict(bias=torch.zeros(200, device="cuda")), dict(score="sigmoid"),
               dict(n_group=4, topk_group=2, group_score="max"), dict(n_group=4, topk_group=2),
               dict(bias=torch.full((200,), -0.0, device="cuda"), score="sigmoid")):
        run_and_check(x, 12, **kw)
    signed = torch.zeros(2, 64, device="cuda")
    signed[0, ::2] = -0.0
    run_and_check(signed, 8)


def test_scores_closer_than_fp32(cuda_device):
    """Biased scores whose 64-bit order fp32 sums cannot tell: 1 + a few 2^-26."""
    t, e = 64, 256
    x = torch.full((t, e), -200.0, device="cuda")
    x[:, 0] = 0.0
    x[:, 64:128] = -18.02 - torch.rand(t, 64, device="cuda") * 0.1      # sigmoid about 2^-26
    bias = torch.ones(e, device="cuda")
    bias[0] = 0.0
    run_and_check(x, 16, bias=bias, score="sigmoid")
    run_and_check(x, 16, bias=bias, score="softmax")
    run_and_check(x, 16, bias=bias, score="sigmoid", n_group=8, topk_group=3)


def test_masked_rows(cuda_device):
    """-inf and NaN logits, rows with fewer live experts than top_k or none, +inf."""
    inf, nan = math.inf, math.nan
    x = logits(8, 48, torch.float32, 9)
    x[1] = -inf
    x[2] = nan
    x[3, 3:] = -inf
    x[4, 5] = inf
    x[5, [7, 40]] = inf
    x[6, ::2] = nan
    x[7] = torch.finfo(torch.float32).min
    bias = torch.zeros(48, device="cuda")
    bias[11], bias[12], bias[13] = -inf, nan, inf
    for score in ("softmax", "sigmoid"):
        for kw in (dict(), dict(bias=bias), dict(n_group=6, topk_group=2), dict(bias=bias, n_group=6, topk_group=2)):
            for renorm in (True, False):
                idx, w = run_and_check(x, 6, score=score, renormalize=renorm, **kw)
                assert w.isfinite().all()
                assert all(len(set(r)) == 6 for r in idx.tolist())
                assert (w[1] == 0).all() and (w[2] == 0).all()


def test_groups_without_the_rows_maximum(cuda_device):
    """Renormalised weights where the kept groups hold only negligible scores."""
    x = torch.full((2, 16), -80.0, device="cuda")
    x[:, 0] = 30.0                     # the best expert is alone in a weak group
    x[:, 8:] = torch.arange(8, device="cuda") - 60.0
    bias = torch.zeros(16, device="cuda")
    bias[8:] = 2.0
    run_and_check(x, 4, n_group=2, topk_group=1, bias=bias)
    run_and_check(x, 4, n_group=2, topk_group=1, bias=bias, renormalize=False)


def test_strides_empty_outputs_stream_and_graph(cuda_device):
    wide = logits(50, 300, torch.float16, 3)
    run_and_check(wide[:, 7:207], 5)
    run_and_check(logits(200, 50, torch.bfloat16, 4).t(), 5)
    idx, w = moe_b200.route_topk(torch.empty(0, 64, device="cuda"), 4)
    assert idx.shape == (0, 4) and w.shape == (0, 4)
    x = logits(50, 64, torch.float32, 5)
    gi, gw = torch.empty(50, 4, dtype=torch.int32, device="cuda"), torch.empty(50, 4, device="cuda")
    oi, ow = moe_b200.route_topk(x, 4, topk_idx=gi, topk_weights=gw)
    assert oi is gi and ow is gw
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gi, gw = moe_b200.route_topk(x, 4)
    x.copy_(logits(50, 64, torch.float32, 6))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        idx, w = run_and_check(x, 4)
    torch.cuda.synchronize()
    assert torch.equal(gi, idx) and torch.equal(gw, w)


def test_same_choice_as_the_fused_router(cuda_device):
    """The layer's own router and the general form agree on its shapes."""
    from gpu_helpers import run_cuda
    shape = workloads.tiny_shape(300)
    inp = workloads.make_inputs(shape, seed=77, device="cuda")
    _, views, _ = run_cuda(inp, shape)
    idx, w = moe_b200.route_topk(inp["routing_logits"], shape.top_k, bias=inp["routing_bias"], score="sigmoid",
                                 n_group=shape.n_group, topk_group=shape.topk_group,
                                 routed_scaling_factor=shape.routed_scaling_factor)
    assert torch.equal(idx, views["topk_idx"])
    assert ((w - views["topk_weights"]).abs() <= 2 ** -20 * w).all()


def test_offsets_past_32_bits(cuda_device):
    t, e = 2 ** 22 + 50, 512
    x = torch.zeros(t, e, dtype=torch.float16, device="cuda")
    x[:, 100] = 1.0
    x[-300:] = logits(300, e, torch.float16, 8)
    idx, w = moe_b200.route_topk(x, 2, renormalize=False)
    assert (idx[:-300] == torch.tensor([100, 0], device="cuda")).all()
    ref_idx, ref_w = reference(x[-300:], 2, renormalize=False)
    assert torch.equal(idx[-300:].cpu().long(), ref_idx)
    assert ((w[-300:].double().cpu() - ref_w).abs() <= ref_w * 2 ** -18).all()
