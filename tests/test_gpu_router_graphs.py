"""Router logits in captured graphs, where a graph keeps the addresses of its scratch."""
import torch
import pytest

import moe_b200
from moe_b200 import api

pytestmark = pytest.mark.gpu


def make(t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(t, 1024, generator=g, device="cuda").to(torch.bfloat16),
            (0.05 * torch.randn(256, 1024, generator=g, device="cuda")).to(torch.bfloat16))


def test_a_graph_has_scratch_of_its_own(cuda_device):
    """The buffer that eager calls share, and replace by a larger one, is no graph's: graphs
    are replayed beside each other and after it is gone."""
    sizes = (300, 700, 1500)
    side = torch.cuda.Stream()
    runs = []
    for i, t in enumerate(sizes):
        x, w = make(t, i)
        want = moe_b200.router_logits(x, w)
        torch.cuda.synchronize()
        before = dict(api._router_ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = moe_b200.router_logits(x, w)
        assert api._router_ws == before
        runs.append((graph, torch.cuda.Stream(), want, out, x, w))
    moe_b200.router_logits(*make(9000, 9))      # the eager calls' buffer grows
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, want, out, *_ in runs:
        assert torch.equal(out, want)
