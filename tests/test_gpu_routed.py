"""The layer with a routing made elsewhere (``run_routed``): bit for bit the
fused layer's result on the same routing, and the oracle's experts on others."""
import numpy as np
import pytest
import torch

import moe_b200
import moe_oracle as mo
from gpu_helpers import run_cuda
from moe_b200 import _lib, api, workloads

pytestmark = pytest.mark.gpu


def layer(inp):
    return [inp[k] for k in ("hidden_states", "hidden_states_scale", "gemm1_weights", "gemm1_weights_scale",
                             "gemm2_weights", "gemm2_weights_scale", "local_expert_offset")]


def empty_out(inp):
    return torch.full(inp["hidden_states"].shape, float("nan"), dtype=torch.bfloat16, device="cuda")


def oracle(inp, idx, w, e_local, offset=0):
    """sum_k w_k E_k(x) over a token's entries, with the oracle's experts."""
    h = mo.to_numpy_inputs({k: v for k, v in inp.items() if isinstance(v, torch.Tensor)})
    idx, w = idx.cpu().numpy(), w.cpu().numpy()
    out = np.zeros(h["hidden_states"].shape, dtype=np.float32)
    for e in range(e_local):
        tok, k = np.nonzero(idx == e + offset)
        if len(tok) == 0:
            continue
        rows = np.unique(tok)
        y = mo.expert_forward(h["hidden_states"][rows], h["hidden_states_scale"][:, rows], h["gemm1_weights"][e],
                              h["gemm1_weights_scale"][e], h["gemm2_weights"][e], h["gemm2_weights_scale"][e],
                              h["gemm1_weights"][e].shape[0] // 2)
        for t, kk in zip(tok, k):
            out[t] += y[np.searchsorted(rows, t)] * w[t, kk]
    return out


def close(out, ref):
    got = out.float().cpu().numpy()
    np.testing.assert_allclose(got, ref, atol=1e-2, rtol=2e-2)
    assert mo.cosine(got, ref) >= 0.9999


@pytest.mark.parametrize("t", [1, 3, 17, 64, 300, 1500])
def test_same_bits_as_the_fused_layer(cuda_device, t):
    shape = workloads.tiny_shape(t)
    inp = workloads.make_inputs(shape, seed=300 + t, device="cuda")
    want = empty_out(inp)
    moe_b200.run(*workloads.run_args(inp), want, n_group=shape.n_group, topk_group=shape.topk_group,
                 top_k=shape.top_k, deterministic=True)
    _, views, _ = run_cuda(inp, shape)
    idx, w = views["topk_idx"].clone(), views["topk_weights"].clone()
    out = empty_out(inp)
    assert moe_b200.run_routed(idx, w, *layer(inp), out, deterministic=True) is None
    assert torch.equal(out, want)
    out = empty_out(inp)
    moe_b200.run_routed(idx, w, *layer(inp), out)
    close(out, want.float().cpu().numpy())


def routing(t, e, k, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return moe_b200.route_topk(torch.randn(t, e, generator=g, device="cuda"), k)


@pytest.mark.parametrize("t,e,k", [(1, 6, 2), (5, 60, 8), (130, 10, 1), (700, 6, 3)])
def test_softmax_routing_over_any_expert_count(cuda_device, t, e, k):
    """Expert counts the fused router does not take."""
    shape = workloads.MoeShape(t=t, hidden=512, inter=256, e_global=e, e_local=e)
    inp = workloads.make_inputs(shape, seed=400 + t, device="cuda")
    idx, w = routing(t, e, k, 500 + t)
    out = empty_out(inp)
    moe_b200.run_routed(idx, w, *layer(inp), out)
    close(out, oracle(inp, idx, w, e))


@pytest.mark.parametrize("t", [4, 200])
def test_padding_repeated_and_foreign_experts(cuda_device, t):
    """Ids outside the experts count for nothing, also with NaN beside them; a
    repeated id counts with the sum of its weights; other shards' experts are left out."""
    shape = workloads.MoeShape(t=t, hidden=512, inter=256, e_global=12, e_local=5, local_expert_offset=4)
    inp = workloads.make_inputs(shape, seed=600 + t, device="cuda")
    idx, w = routing(t, 12, 4, 700 + t)
    idx[0] = -1
    idx[1] = torch.tensor([5, 5, 5, 5], dtype=torch.int32)
    idx[2] = torch.tensor([4, 12, 4, 2 ** 31 - 1], dtype=torch.int32)
    idx[3] = torch.tensor([-(2 ** 31), 8, 3, 8], dtype=torch.int32)
    ref = oracle(inp, idx, w, 5, 4)
    w[0] = float("nan")
    w[2, [1, 3]] = float("inf")
    for det in (True, False):
        out = empty_out(inp)
        moe_b200.run_routed(idx, w, *layer(inp), out, num_experts=12, deterministic=det)
        close(out, ref)
        assert (out[0] == 0).all()


def test_shared_expert_empty_batch_and_graph(cuda_device):
    shape = workloads.MoeShape(t=70, hidden=512, inter=256, e_global=8, e_local=8)
    inp = workloads.make_inputs(shape, seed=800, device="cuda")
    idx, w = routing(70, 7, 3, 801)     # the last slice is the shared expert's
    out = empty_out(inp)
    moe_b200.run_routed(idx, w, *layer(inp), out, n_shared_experts=1)
    with_shared = torch.cat([idx, torch.full_like(idx[:, :1], 7)], 1), torch.cat([w, torch.ones_like(w[:, :1])], 1)
    ref = oracle(inp, *with_shared, 8)
    close(out, ref)
    moe_b200.run_routed(idx[:0], w[:0], *[v[:0] if i == 0 else v[:, :0] if i == 1 else v
                                          for i, v in enumerate(layer(inp))], out[:0])
    ws = torch.empty(1 << 25, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    out2 = empty_out(inp)
    with torch.cuda.graph(graph):
        moe_b200.run_routed(idx, w, *layer(inp), out2, n_shared_experts=1, workspace=ws, deterministic=True)
    w.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    ref = oracle(inp, with_shared[0], torch.cat([w, torch.ones_like(w[:, :1])], 1), 8)
    close(out2, ref)


def test_graphs_replayed_at_the_same_time(cuda_device):
    """Graphs captured without a workspace of the caller's do not share scratch."""
    shape = workloads.MoeShape(t=300, hidden=512, inter=256, e_global=10, e_local=10)
    inp = workloads.make_inputs(shape, seed=900, device="cuda")
    runs = []
    for i in range(3):
        idx, w = routing(300, 10, 3, 901 + i)
        want, out = empty_out(inp), empty_out(inp)
        moe_b200.run_routed(idx, w, *layer(inp), want, deterministic=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            moe_b200.run_routed(idx, w, *layer(inp), out, deterministic=True)
        runs.append((graph, torch.cuda.Stream(), want, out, idx, w))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, want, out, *_ in runs:
        assert torch.equal(out, want)


def test_refusals(cuda_device):
    shape = workloads.tiny_shape(4)
    inp = workloads.make_inputs(shape, seed=1, device="cuda")
    out = empty_out(inp)
    idx = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    w = torch.ones(4, 4, device="cuda")
    for a, b in ((idx.long(), w), (idx, w.double()), (idx[:3], w[:3]), (idx, w[:, :2]), (idx[0], w[0]),
                 (idx.repeat(1, 3), w.repeat(1, 3)), (idx[:, :0], w[:, :0])):
        with pytest.raises(AssertionError):
            moe_b200.run_routed(a, b, *layer(inp), out)
    with pytest.raises(AssertionError):
        moe_b200.run_routed(idx, w, *layer(inp), out, num_experts=257)
    with pytest.raises(AssertionError):
        moe_b200.run_routed(idx, w, *layer(inp), out, workspace=torch.empty(1 << 24, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        moe_b200.run_routed(idx, w, *layer(inp), out, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    with pytest.raises(AssertionError):
        moe_b200.run_routed(idx, w, *layer(inp), out, num_experts=15)
    args, keep, _ = api.build_args(*workloads.run_args(inp), out, shape.n_group, shape.topk_group, shape.top_k)
    lib = _lib.load()
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    assert lib.moe_fp8_forward_routed(args, idx.data_ptr(), w.data_ptr(), None) == _lib.MOE_ERR_SHAPE
    args.n_group = args.topk_group = 0
    assert lib.moe_fp8_forward(args, None) == _lib.MOE_ERR_SHAPE
    args.flags = _lib.MOE_FLAG_DEBUG
    assert lib.moe_fp8_forward_routed(args, idx.data_ptr(), w.data_ptr(), None) == _lib.MOE_ERR_INVALID_ARG
