"""The first call of a process inside a graph capture: what a product or the layer sets
up once for a device is allowed there."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
sys.path[:0] = {path!r}
import torch, moe_b200
x = torch.randn({t}, 512, device="cuda").to(torch.bfloat16)
codes = torch.randint(0, 256, (300, 256), dtype=torch.uint8, device="cuda")
scales = torch.full(moe_b200.fp4_scales_shape(300, 512), 48, dtype=torch.uint8, device="cuda")
def call():
    q, s, y, _ = moe_b200.rms_norm_quantize_1x128(x, torch.ones_like(x[0]), normed=True)
    return moe_b200.linear_fp4(y, codes, scales)
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    x.normal_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call()) and out.isfinite().all()
print("same")
"""


@pytest.mark.parametrize("t", [3, 50, 900])
def test_captured(cuda_device, t):
    p = subprocess.run([sys.executable, "-c", PROGRAM.format(path=sys.path, t=t)], capture_output=True, text=True,
                       timeout=300)
    assert p.returncode == 0 and p.stdout.strip() == "same", p.stderr[-2000:]
