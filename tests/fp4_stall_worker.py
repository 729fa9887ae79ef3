"""4-bit products whose first wait runs out (MOE_FP4_TEST_STALL), in a process of its own:
prints one JSON line with what each gave.  Run by test_gpu_fp4_failure.py."""
import json
import os
import sys
import time

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "mlsys26-flashinfer-moe_b200"))
import torch  # noqa: E402

import moe_b200  # noqa: E402
from moe_b200 import _lib  # noqa: E402


def stalled(x, w, fmt, quantised):
    """One product on the current stream with the hook set, tokens quantised before or on the way."""
    t, k = x.shape
    n = w[0].shape[0]
    out = torch.zeros(t, n, dtype=torch.float32, device="cuda")
    code = (_lib.MOE_MXFP4 if fmt == "mxfp4" else _lib.MOE_NVFP4) | _lib.MOE_FP4_TEST_STALL
    stream = torch.cuda.current_stream().cuda_stream
    lib = _lib.load()
    if quantised:
        c, s = moe_b200.quantize_fp4(x, fmt)
        st = lib.moe_fp4_matmul(c.data_ptr(), k // 2, s.data_ptr(), None, w[0].data_ptr(), k // 2, w[1].data_ptr(), None,
                                code, t, n, k, out.data_ptr(), _lib.MOE_F32, n, stream)
    else:
        ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
        st = lib.moe_fp4_linear(x.data_ptr(), _lib.MOE_BF16, k, None, w[0].data_ptr(), k // 2, w[1].data_ptr(), None,
                                code, t, n, k, out.data_ptr(), _lib.MOE_F32, n, ws.data_ptr(), ws.numel(), stream)
    torch.cuda.synchronize()
    return st, out


def main():
    gen = torch.Generator(device="cuda").manual_seed(3)
    results = []
    for t, n, k, quantised in json.loads(sys.argv[1]):
        for fmt in ("nvfp4", "mxfp4"):
            x = torch.randn(t, k, generator=gen, device="cuda").to(torch.bfloat16)
            w = moe_b200.quantize_fp4(torch.randn(n, k, generator=gen, device="cuda"), fmt)
            want = moe_b200.linear_fp4(x, *w, fmt, dtype=torch.float32)
            torch.cuda.synchronize()
            began = time.monotonic()
            st, out = stalled(x, w, fmt, quantised)
            took = time.monotonic() - began
            after = moe_b200.linear_fp4(x, *w, fmt, dtype=torch.float32)
            results.append(dict(case=[t, n, k, fmt], status=st, nan=out.isnan().all().item(), seconds=took,
                                after=torch.equal(after, want)))
    print(json.dumps(dict(results=results, error=moe_b200.fp4_device_error())))


if __name__ == "__main__":
    main()
