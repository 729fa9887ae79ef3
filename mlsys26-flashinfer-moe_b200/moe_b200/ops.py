"""The operators around the layer: what comes before and beside ``run()`` in a
transformer block.

* ``rms_norm_quantize_1x128``  residual addition, RMS norm and the FP8
  quantisation that ``run()`` takes, in one pass;
* ``route_topk``  routing to experts with softmax or sigmoid scores, for
  ``run_routed()``;
* ``quantize_fp4`` / ``dequantize_fp4`` / ``matmul_fp4`` / ``linear_fp4``
  microscaled 4-bit matrices and their product, for the dense projections.

All run on the current stream of their tensors' device (whichever device is
current), without synchronising; inference only (no gradients).  Shape and type
errors raise ``AssertionError``, like ``run()``'s.  Inputs that are not on the
GPU, or whose rows are not contiguous and 16-byte aligned, are not accepted
silently: the former raise, the latter are copied.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .api import _F8, _raise

_DTYPES = {torch.float32: _lib.MOE_F32, torch.bfloat16: _lib.MOE_BF16, torch.float16: _lib.MOE_F16}
_HALF = (torch.bfloat16, torch.float16)
_SCORES = {"softmax": _lib.MOE_SCORE_SOFTMAX, "sigmoid": _lib.MOE_SCORE_SIGMOID}
_GROUP_SCORES = {"top2": _lib.MOE_GROUP_TOP2, "max": _lib.MOE_GROUP_MAX}
_FORMATS = {"mxfp4": _lib.MOE_MXFP4, "nvfp4": _lib.MOE_NVFP4}
_RUN = {"mxfp4": 32, "nvfp4": 16}


def _call(name: str, device: torch.device, *args) -> None:
    """One C entry point on the current stream of ``device``."""
    fn = getattr(_lib.load(), name)
    index = device.index
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == index:
        code = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, stream)
    if code:
        _raise(code, name)


def _on_gpu(device: Optional[torch.device], **tensors) -> torch.device:
    """All tensors (``None`` is skipped) are on one CUDA device; returns it."""
    for name, t in tensors.items():
        if t is None:
            continue
        assert t.is_cuda, f"{name} must be a CUDA tensor"
        if device is None:
            device = t.device
        assert t.device == device, f"{name} must be on {device}"
    return device


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows the kernels can read: unit column stride, 16-byte aligned
    rows that do not overlap; otherwise a contiguous copy."""
    size = t.element_size()
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and \
            (t.shape[0] == 1 or (t.stride(0) * size % 16 == 0 and t.stride(0) >= t.shape[1])):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ld(t: torch.Tensor) -> int:
    """Row stride; that of a single row may be anything and is not used."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _out_rows(t: torch.Tensor, name: str, shape, dtype) -> torch.Tensor:
    assert tuple(t.shape) == tuple(shape) and t.dtype == dtype, f"{name} must be {dtype} {list(shape)}"
    assert t.shape[0] == 0 or (t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (
        t.shape[0] == 1 or (t.stride(0) * t.element_size() % 16 == 0 and t.stride(0) >= t.shape[1]))), \
        f"{name} must have contiguous, 16-byte aligned rows"
    return t


def rms_norm_quantize_1x128(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                            residual: Optional[torch.Tensor] = None,
                            residual_out: Optional[torch.Tensor] = None,
                            normed: Union[bool, torch.Tensor] = False,
                            q: Optional[torch.Tensor] = None,
                            scale: Optional[torch.Tensor] = None
                            ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor],
                                       Optional[torch.Tensor]]:
    """``h = x + residual``, ``y = h * rsqrt(mean(h^2) + eps) * weight`` and the
    FP8 form of ``y``; returns ``(q, scale, normed, residual_out)``.

    ``x`` ``[T, H]`` is bf16 or fp16, ``H`` a multiple of 128; ``weight`` ``[H]``
    and ``residual`` ``[T, H]`` are of ``x``'s type or fp32.  ``q`` (e4m3 ``[T,
    H]``) and ``scale`` (fp32 ``[H/128, T]``) are what ``run()`` takes as
    ``hidden_states`` / ``hidden_states_scale``, quantised from the unrounded
    ``y`` (``scale = max(amax/448, 1e-12)`` per token and 128 columns).
    ``normed=True`` (or a tensor to write) also gives ``y`` in ``x``'s type, for
    ``router_logits``; otherwise ``None``.  ``residual_out`` receives ``h`` in
    the residual's type (``residual`` itself: in place); ``None`` without a
    residual.
    """
    assert x.dim() == 2 and x.dtype in _HALF, "x must be a bf16 or fp16 [T, H] tensor"
    t, h = x.shape
    assert h >= 128 and h % 128 == 0, "H must be a multiple of 128"
    assert weight.shape == (h,) and weight.dtype in (x.dtype, torch.float32), \
        f"weight must be {x.dtype} or float32 [{h}]"
    assert residual is not None or residual_out is None, "residual_out needs a residual"
    device = _on_gpu(x.device, x=x, weight=weight, residual=residual, residual_out=residual_out,
                     normed=normed if isinstance(normed, torch.Tensor) else None, q=q, scale=scale)
    x = _rows(x)
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.contiguous().clone()
    r_ptr = ro_ptr = n_ptr = None
    r_dtype, ld_r, ld_ro, ld_n = _DTYPES[x.dtype], h, h, h
    if residual is not None:
        assert residual.shape == (t, h) and residual.dtype in (x.dtype, torch.float32), \
            f"residual must be {x.dtype} or float32 [{t}, {h}]"
        r_dtype = _DTYPES[residual.dtype]
        if residual_out is None:
            residual_out = torch.empty(t, h, dtype=residual.dtype, device=device)
        else:
            _out_rows(residual_out, "residual_out", (t, h), residual.dtype)
        residual = _rows(residual)
        r_ptr, ld_r = residual.data_ptr(), _ld(residual)
        ro_ptr, ld_ro = residual_out.data_ptr(), _ld(residual_out)
    if normed is True:
        normed = torch.empty(t, h, dtype=x.dtype, device=device)
    elif normed is False:
        normed = None
    if normed is not None:
        _out_rows(normed, "normed", (t, h), x.dtype)
        n_ptr, ld_n = normed.data_ptr(), _ld(normed)
    if q is None:
        q = torch.empty(t, h, dtype=_F8, device=device)
    else:
        assert q.shape == (t, h) and q.dtype == _F8 and q.is_contiguous(), f"q must be e4m3 [{t}, {h}]"
    if scale is None:
        scale = torch.empty(h // 128, t, dtype=torch.float32, device=device)
    else:
        assert scale.shape == (h // 128, t) and scale.dtype == torch.float32 and \
            scale.is_contiguous(), f"scale must be float32 [{h // 128}, {t}]"
    _call("moe_rms_norm_1x128", device, x.data_ptr(), _DTYPES[x.dtype], _ld(x), r_ptr, r_dtype, ld_r,
          weight.data_ptr(), _DTYPES[weight.dtype], eps, t, h, ro_ptr, ld_ro, n_ptr, ld_n,
          q.data_ptr(), scale.data_ptr())
    return q, scale, normed, residual_out


def route_topk(logits: torch.Tensor, top_k: int, *, bias: Optional[torch.Tensor] = None,
               score: str = "softmax", n_group: int = 1, topk_group: int = 1,
               group_score: str = "top2", renormalize: bool = True,
               routed_scaling_factor: float = 1.0, topk_idx: Optional[torch.Tensor] = None,
               topk_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Routing to experts; returns ``(topk_idx int32, topk_weights fp32)``, both
    ``[T, top_k]``, for ``run_routed()``.

    ``s`` is the softmax or sigmoid (``score``) of ``logits`` ``[T, E]`` (fp32,
    bf16 or fp16, ``E <= 1024``); ``c = s + bias`` (``[E]``) decides: of the
    ``n_group`` equal runs of experts the ``topk_group`` with the largest best
    ``c`` (``group_score="max"``) or sum of the two largest (``"top2"``) are kept,
    then the ``top_k <= 32`` largest ``c`` in them are taken, largest first, ties
    to the lowest id.  The weights are ``s`` there, divided by their sum (plus
    1e-20) if ``renormalize``, times ``routed_scaling_factor``.  The order is
    that of the exact scores.  NaN logits and biases count as ``-inf``: such
    experts rank last; a ``-inf`` logit weighs 0, also in a row of nothing else.
    """
    assert logits.dim() == 2 and logits.dtype in _DTYPES, "logits must be fp32, bf16 or fp16 [T, E]"
    assert score in _SCORES, "score must be 'softmax' or 'sigmoid'"
    assert group_score in _GROUP_SCORES, "group_score must be 'top2' or 'max'"
    t, e = logits.shape
    top_k = int(top_k)
    device = _on_gpu(logits.device, logits=logits, bias=bias, topk_idx=topk_idx,
                     topk_weights=topk_weights)
    if logits.stride(1) != 1 or (t > 1 and logits.stride(0) < e):
        logits = logits.contiguous()
    b_ptr, b_dtype = None, _lib.MOE_F32
    if bias is not None:
        assert bias.shape == (e,) and bias.dtype in _DTYPES, f"bias must be fp32, bf16 or fp16 [{e}]"
        bias = bias.contiguous()
        b_ptr, b_dtype = bias.data_ptr(), _DTYPES[bias.dtype]
    if topk_idx is None:
        topk_idx = torch.empty(t, max(top_k, 0), dtype=torch.int32, device=device)
    if topk_weights is None:
        topk_weights = torch.empty(t, max(top_k, 0), dtype=torch.float32, device=device)
    assert topk_idx.shape == (t, top_k) and topk_idx.dtype == torch.int32 and \
        topk_idx.is_contiguous(), f"topk_idx must be int32 [{t}, {top_k}]"
    assert topk_weights.shape == (t, top_k) and topk_weights.dtype == torch.float32 and \
        topk_weights.is_contiguous(), f"topk_weights must be float32 [{t}, {top_k}]"
    _call("moe_route_topk", device, logits.data_ptr(), _DTYPES[logits.dtype], _ld(logits), b_ptr,
          b_dtype, t, e, top_k, _SCORES[score], int(n_group), int(topk_group),
          _GROUP_SCORES[group_score], 1 if renormalize else 0, routed_scaling_factor,
          topk_idx.data_ptr(), topk_weights.data_ptr())
    return topk_idx, topk_weights


def fp4_scales_shape(rows: int, k: int, fmt: str = "nvfp4") -> Tuple[int, int, int, int, int]:
    """Shape ``[ceil(R/128), ceil(runs/4), 32, 4, 4]`` of a matrix's scales: the
    scale of row ``r`` and run ``b`` (16 or 32 columns) is element
    ``[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]``."""
    assert fmt in _FORMATS, "fmt must be 'mxfp4' or 'nvfp4'"
    per = 4 * _RUN[fmt]
    return (rows + 127) // 128, (k + per - 1) // per, 32, 4, 4


def _check_format(fmt: str, **global_scales) -> int:
    assert fmt in _FORMATS, "fmt must be 'mxfp4' or 'nvfp4'"
    for name, g in global_scales.items():
        if g is not None:
            assert fmt == "nvfp4", f"{name} belongs to nvfp4"
            assert g.dtype == torch.float32 and g.numel() == 1, f"{name} must be one float32"
    return _FORMATS[fmt]


def _check_matrix(codes: torch.Tensor, scales: torch.Tensor, fmt: str, name: str):
    assert codes.dim() == 2 and codes.dtype == torch.uint8, f"{name}_codes must be uint8 [rows, K/2]"
    r, k = codes.shape[0], 2 * codes.shape[1]
    assert k >= 32 and k % 32 == 0, "K must be a multiple of 32"
    shape = fp4_scales_shape(r, k, fmt)
    assert scales.dtype == torch.uint8 and tuple(scales.shape) == shape, \
        f"{name}_scales must be uint8 {list(shape)} (fp4_scales_shape)"
    assert scales.is_contiguous() and scales.data_ptr() % 16 == 0, \
        f"{name}_scales must be contiguous and 16-byte aligned"
    return r, k


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def quantize_fp4(x: torch.Tensor, fmt: str = "nvfp4", *, global_scale: Optional[torch.Tensor] = None,
                 codes: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` ``[R, K]`` (fp32, bf16 or fp16, ``K`` a multiple of 32) in microscaled
    4 bits: ``(codes uint8 [R, K/2], scales uint8 fp4_scales_shape(R, K, fmt))``.

    ``"mxfp4"``: a power-of-two scale (e8m0) for 32 columns,
    ``2^(floor(log2(amax)) - 2)``.  ``"nvfp4"``: an e4m3 scale for 16 columns,
    ``amax / (6 * global_scale)``, with ``global_scale`` one fp32 on the device
    (default 1; ``amax of the tensor / 2688`` uses the whole range).  A code is
    ``x / (scale * global_scale)`` rounded to e2m1, even columns in the low
    half of a byte.  Runs with a NaN or infinity get a NaN scale.
    """
    f = _check_format(fmt, global_scale=global_scale)
    assert x.dim() == 2 and x.dtype in _DTYPES, "x must be fp32, bf16 or fp16 [R, K]"
    r, k = x.shape
    assert k >= 32 and k % 32 == 0, "K must be a multiple of 32"
    device = _on_gpu(x.device, x=x, global_scale=global_scale, codes=codes, scales=scales)
    x = _rows(x)
    if codes is None:
        codes = torch.empty(r, k // 2, dtype=torch.uint8, device=device)
    if scales is None:
        scales = torch.empty(fp4_scales_shape(r, k, fmt), dtype=torch.uint8, device=device)
    assert codes.is_contiguous(), "codes must be contiguous"
    assert _check_matrix(codes, scales, fmt, "output") == (r, k), f"codes must be uint8 [{r}, {k // 2}]"
    _call("moe_fp4_quantize", device, x.data_ptr(), _DTYPES[x.dtype], _ld(x), r, k, f, _ptr(global_scale),
          codes.data_ptr(), scales.data_ptr())
    return codes, scales


def dequantize_fp4(codes: torch.Tensor, scales: torch.Tensor, fmt: str = "nvfp4", *,
                   global_scale: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values ``[R, K]`` of a matrix in microscaled 4 bits, rounded to ``dtype``."""
    f = _check_format(fmt, global_scale=global_scale)
    r, k = _check_matrix(codes, scales, fmt, "input")
    assert dtype in _DTYPES, "dtype must be fp32, bf16 or fp16"
    device = _on_gpu(codes.device, codes=codes, scales=scales, global_scale=global_scale, out=out)
    codes = _rows(codes)
    if out is None:
        out = torch.empty(r, k, dtype=dtype, device=device)
    assert out.shape == (r, k) and out.dtype == dtype and out.is_contiguous(), \
        f"out must be a contiguous {dtype} [{r}, {k}]"
    _call("moe_fp4_dequantize", device, codes.data_ptr(), _ld(codes), scales.data_ptr(), r, k, f,
          _ptr(global_scale), out.data_ptr(), _DTYPES[dtype])
    return out


def _product_out(out: Optional[torch.Tensor], t: int, n: int, dtype: torch.dtype,
                 device: torch.device) -> torch.Tensor:
    assert dtype in _DTYPES, "dtype must be fp32, bf16 or fp16"
    if out is None:
        return torch.empty(t, n, dtype=dtype, device=device)
    assert out.shape == (t, n) and out.dtype == dtype, f"out must be {dtype} [{t}, {n}]"
    assert out.device == device, f"out must be on {device}"
    assert t == 0 or n == 1 or out.stride(1) == 1, "out must have contiguous rows"
    assert t <= 1 or out.stride(0) >= n, "rows of out must not overlap"
    return out


def matmul_fp4(a_codes: torch.Tensor, a_scales: torch.Tensor, b_codes: torch.Tensor,
               b_scales: torch.Tensor, fmt: str = "nvfp4", *,
               a_global_scale: Optional[torch.Tensor] = None,
               b_global_scale: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.bfloat16,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``A [T, K] . B [N, K]^T`` of two matrices in microscaled 4 bits, summed in
    fp32 on the tensor core and rounded once to ``dtype``.  Bit-identical from
    run to run."""
    f = _check_format(fmt, a_global_scale=a_global_scale, b_global_scale=b_global_scale)
    t, k = _check_matrix(a_codes, a_scales, fmt, "a")
    n, kb = _check_matrix(b_codes, b_scales, fmt, "b")
    assert k == kb, f"a and b must have the same K, not {k} and {kb}"
    device = _on_gpu(a_codes.device, a_codes=a_codes, a_scales=a_scales, b_codes=b_codes,
                     b_scales=b_scales, a_global_scale=a_global_scale, b_global_scale=b_global_scale)
    a_codes, b_codes = _rows(a_codes), _rows(b_codes)
    out = _product_out(out, t, n, dtype, device)
    _call("moe_fp4_matmul", device, a_codes.data_ptr(), _ld(a_codes), a_scales.data_ptr(),
          _ptr(a_global_scale), b_codes.data_ptr(), _ld(b_codes), b_scales.data_ptr(),
          _ptr(b_global_scale), f, t, n, k, out.data_ptr(), _DTYPES[dtype], _ld(out))
    return out


def linear_fp4(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor, fmt: str = "nvfp4", *,
               x_global_scale: Optional[torch.Tensor] = None,
               w_global_scale: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [T, K] . W [N, K]^T`` with ``W`` in microscaled 4 bits: quantises ``x``
    (fp32, bf16 or fp16) as ``quantize_fp4`` does and multiplies as
    ``matmul_fp4`` does, in ``dtype`` (default: ``x``'s)."""
    f = _check_format(fmt, x_global_scale=x_global_scale, w_global_scale=w_global_scale)
    assert x.dim() == 2 and x.dtype in _DTYPES, "x must be fp32, bf16 or fp16 [T, K]"
    n, k = _check_matrix(w_codes, w_scales, fmt, "w")
    t = x.shape[0]
    assert x.shape[1] == k, f"x must be [T, {k}]"
    device = _on_gpu(x.device, x=x, w_codes=w_codes, w_scales=w_scales, x_global_scale=x_global_scale,
                     w_global_scale=w_global_scale)
    x, w_codes = _rows(x), _rows(w_codes)
    dtype = x.dtype if dtype is None else dtype
    out = _product_out(out, t, n, dtype, device)
    # codes and scales of x live for this call only: a buffer of the current
    # stream (or of the graph being captured), never shared between calls
    shape = fp4_scales_shape(t, k, fmt)
    nbytes = (t * (k // 2) + 255) // 256 * 256 + shape[0] * shape[1] * 512
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call("moe_fp4_linear", device, x.data_ptr(), _DTYPES[x.dtype], _ld(x), _ptr(x_global_scale),
          w_codes.data_ptr(), _ld(w_codes), w_scales.data_ptr(), _ptr(w_global_scale), f, t, n, k,
          out.data_ptr(), _DTYPES[dtype], _ld(out), ws.data_ptr(), nbytes)
    return out


def fp4_device_error(device: Optional[torch.device] = None) -> Tuple[int, int]:
    """(code, info) of the first device-side wait of a 4-bit product that ran out
    on ``device`` since the library was loaded; (0, 0) if none.  Blocks."""
    code, info = ctypes.c_int32(0), ctypes.c_int32(0)
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream().cuda_stream
        st = _lib.load().moe_fp4_device_error(stream, ctypes.byref(code), ctypes.byref(info))
    if st:
        _raise(st, "moe_fp4_device_error")
    return code.value, info.value
