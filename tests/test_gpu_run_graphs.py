"""run() in captured graphs, where a graph keeps the addresses of its workspace."""
import pytest
import torch

import moe_b200
from moe_b200 import api, workloads

pytestmark = pytest.mark.gpu


def test_a_graph_has_a_workspace_of_its_own(cuda_device):
    """The workspace that eager calls share, and replace by a larger one, is no graph's:
    graphs are replayed beside each other and after it is gone."""
    side = torch.cuda.Stream()
    runs = []

    def call(shape, inp, out):
        moe_b200.run(*workloads.run_args(inp), out, n_group=shape.n_group, topk_group=shape.topk_group,
                     top_k=shape.top_k, deterministic=True)

    for i, t in enumerate((3, 60, 300, 300)):
        shape = workloads.tiny_shape(t)
        inp = workloads.make_inputs(shape, seed=950 + i, device="cuda")
        want = torch.empty(t, shape.hidden, dtype=torch.bfloat16, device="cuda")
        out = torch.full_like(want, float("nan"))
        call(shape, inp, want)
        torch.cuda.synchronize()
        before = dict(api._workspaces)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(shape, inp, out)
        assert api._workspaces == before
        runs.append((graph, torch.cuda.Stream(), want, out, inp))
    shape = workloads.tiny_shape(3000)
    call(shape, workloads.make_inputs(shape, seed=1, device="cuda"),
         torch.empty(3000, shape.hidden, dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, want, out, _ in runs:
        assert torch.equal(out, want)
