"""B200-native (sm_100a) fused FP8 block-scale DeepSeek-V3 MoE forward.

``moe_b200.run`` is a drop-in for ``run()`` of nikhilnd/mlsys26-flashinfer-moe
(``kernel.py:562``); the kernels live in ``libmoe_b200.so`` (C ABI in
``include/moe_b200.h``).
"""
from .api import (run, build_args, forward_args, workspace_views, device_error,  # noqa: F401
                  quantize_1x128, prepare_gemm2_weights, check_workspace, describe_error,
                  raise_device_error, router_logits)
from .api import run_routed  # noqa: F401
from .ops import (rms_norm_quantize_1x128, route_topk, quantize_fp4, dequantize_fp4,  # noqa: F401
                  matmul_fp4, linear_fp4, fp4_scales_shape, fp4_device_error)
from .graph import LayerGraph  # noqa: F401
from . import workloads  # noqa: F401

__all__ = ["run", "build_args", "forward_args", "workspace_views", "device_error", "quantize_1x128",
           "prepare_gemm2_weights", "check_workspace", "describe_error", "raise_device_error",
           "router_logits", "run_routed", "rms_norm_quantize_1x128", "route_topk", "quantize_fp4",
           "dequantize_fp4", "matmul_fp4", "linear_fp4", "fp4_scales_shape", "fp4_device_error",
           "LayerGraph", "workloads"]
