"""The operators around the layer: what comes before and beside ``run()`` in a
transformer block.

* ``rms_norm_quantize_1x128``  residual addition, RMS norm and the FP8
  quantisation that ``run()`` takes, in one pass;
* ``route_topk``  routing to experts with softmax or sigmoid scores, for
  ``run_routed()`` or another expert layer;
* ``quantize_fp4`` / ``dequantize_fp4`` / ``matmul_fp4`` / ``linear_fp4``
  microscaled 4-bit matrices and their product, for the dense projections.

All run on the current stream of their tensors' device (whichever device is
current), without synchronising; inference only (no gradients).  Shape and type
errors raise ``AssertionError``, like ``run()``'s.  Inputs that are not on the
GPU raise as well; those whose rows are not contiguous and 16-byte aligned are
copied.  Outputs must not overlap inputs unless an operator says so.
"""
from __future__ import annotations

import ctypes
import functools
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


_entry: dict = {}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # none without CUDA
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_empty = torch.empty


def _call(name: str, index: int, *args) -> None:
    """One C entry point on the current stream of CUDA device ``index``."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load(), name)
    stream = _raw_stream(index)
    if _current_device() == index:
        code = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, stream)
    if code:
        _raise(code, name)


def _gpu(t: torch.Tensor, name: str) -> int:
    """The CUDA device index of ``t``."""
    assert t.is_cuda, f"{name} must be a CUDA tensor"
    return t.get_device()


def _same(t: Optional[torch.Tensor], name: str, index: int) -> None:
    assert t is None or t.get_device() == index, f"{name} must be on cuda:{index}"


def _rows_ok(t: torch.Tensor) -> bool:
    """Unit column stride and 16-byte aligned rows that do not overlap (the row
    stride of a single row does not matter, a contiguous row of a multiple of
    16 bytes keeps the next one aligned)."""
    if t.data_ptr() % 16:
        return False
    row = t.shape[1] * t.element_size()
    if row % 16 == 0 and t.is_contiguous():
        return True
    ld, col = t.stride()
    return col == 1 and (t.shape[0] == 1 or (ld * t.element_size() % 16 == 0 and ld >= t.shape[1]))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a contiguous copy if its rows are not as the kernels read them."""
    if _rows_ok(t):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ld(t: torch.Tensor) -> int:
    """Row stride; that of a single row may be anything and is not used."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_out(t: torch.Tensor, name: str, shape, dtype, index: int) -> None:
    assert t.shape == shape and t.dtype == dtype, f"{name} must be {dtype} {list(shape)}"
    assert t.get_device() == index, f"{name} must be on cuda:{index}"


def _out_rows(t: torch.Tensor, name: str, shape, dtype, index: int) -> None:
    _check_out(t, name, shape, dtype, index)
    assert t.shape[0] == 0 or _rows_ok(t), f"{name} must have contiguous, 16-byte aligned rows"


def _out_flat(t: torch.Tensor, name: str, shape, dtype, index: int) -> None:
    _check_out(t, name, shape, dtype, index)
    assert t.is_contiguous(), f"{name} must be contiguous"


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
    ``normed=True`` (or a tensor to write) also gives ``y`` in ``x``'s type, in bf16 the
    input of ``router_logits``; otherwise ``None``.  ``residual_out`` receives ``h`` in
    the residual's type (``residual`` itself: in place); ``None`` without a
    residual.
    """
    dtype = x.dtype
    assert x.dim() == 2 and dtype in _HALF, "x must be a bf16 or fp16 [T, H] tensor"
    shape = x.shape
    t, h = shape
    assert h >= 128 and h % 128 == 0, "H must be a multiple of 128"
    assert weight.shape == (h,) and weight.dtype in (dtype, torch.float32), \
        f"weight must be {dtype} or float32 [{h}]"
    assert residual is not None or residual_out is None, "residual_out needs a residual"
    dev, device = _gpu(x, "x"), x.device
    _same(weight, "weight", dev)
    x = _rows(x)
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.contiguous().clone()
    code = _DTYPES[dtype]
    r_ptr = ro_ptr = n_ptr = None
    r_code, ld_r, ld_ro, ld_n = code, h, h, h
    if residual is not None:
        r_dtype = residual.dtype
        assert residual.shape == shape and r_dtype in (dtype, torch.float32), \
            f"residual must be {dtype} or float32 [{t}, {h}]"
        _same(residual, "residual", dev)
        if residual_out is None:
            residual_out = _empty(t, h, dtype=r_dtype, device=device)
        else:
            _out_rows(residual_out, "residual_out", shape, r_dtype, dev)
        residual = _rows(residual)
        r_code, r_ptr, ld_r = _DTYPES[r_dtype], residual.data_ptr(), _ld(residual)
        ro_ptr, ld_ro = residual_out.data_ptr(), _ld(residual_out)
    if normed is False:
        normed = None
    elif normed is True:
        normed = _empty(t, h, dtype=dtype, device=device)
        n_ptr = normed.data_ptr()
    elif normed is not None:
        _out_rows(normed, "normed", shape, dtype, dev)
        n_ptr, ld_n = normed.data_ptr(), _ld(normed)
    if q is None:
        q = _empty(t, h, dtype=_F8, device=device)
    else:
        _out_flat(q, "q", shape, _F8, dev)
    if scale is None:
        scale = _empty(h // 128, t, dtype=torch.float32, device=device)
    else:
        _out_flat(scale, "scale", (h // 128, t), torch.float32, dev)
    _call("moe_rms_norm_1x128", dev, x.data_ptr(), code, _ld(x), r_ptr, r_code, ld_r,
          weight.data_ptr(), _DTYPES[weight.dtype], eps, t, h, ro_ptr, ld_ro, n_ptr, ld_n,
          q.data_ptr(), scale.data_ptr())
    return q, scale, normed, residual_out


def route_topk(logits: torch.Tensor, top_k: int, *, bias: Optional[torch.Tensor] = None,
               score: str = "softmax", n_group: int = 1, topk_group: int = 1,
               group_score: str = "top2", renormalize: bool = True,
               routed_scaling_factor: float = 1.0, topk_idx: Optional[torch.Tensor] = None,
               topk_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Routing to experts; returns ``(topk_idx int32, topk_weights fp32)``, both
    ``[T, top_k]``: what ``run_routed()`` takes, up to its 256 experts and top_k of 8
    (beyond that they are for expert layers of the caller's).

    ``s`` is the softmax or sigmoid (``score``) of ``logits`` ``[T, E]`` (fp32,
    bf16 or fp16, ``E <= 1024``); ``c = s + bias`` (``[E]``) decides: of the
    ``n_group`` equal runs of experts the ``topk_group`` with the largest best
    ``c`` (``group_score="max"``) or sum of the two largest (``"top2"``) are kept,
    then the ``top_k <= 32`` largest ``c`` in them are taken, largest first, ties
    to the lowest id.  The weights are ``s`` there, divided by their sum (plus
    1e-20) if ``renormalize``, times ``routed_scaling_factor``.  The order is
    that of the exact scores.  NaN logits and biases count as ``-inf``.  A ``-inf``
    logit has the score 0: it weighs 0, also in a row of nothing else, and ranks last
    without a bias, with one where that puts it.  A ``-inf`` bias ranks last.
    """
    assert logits.dim() == 2 and logits.dtype in _DTYPES, "logits must be fp32, bf16 or fp16 [T, E]"
    assert score in _SCORES, "score must be 'softmax' or 'sigmoid'"
    assert group_score in _GROUP_SCORES, "group_score must be 'top2' or 'max'"
    t, e = logits.shape
    top_k = int(top_k)
    assert 1 <= top_k <= 32, "top_k must be 1 to 32"
    dev = _gpu(logits, "logits")
    if not logits.is_contiguous() and (logits.stride(1) != 1 or (t > 1 and logits.stride(0) < e)):
        logits = logits.contiguous()
    b_ptr, b_code = None, _lib.MOE_F32
    if bias is not None:
        assert bias.shape == (e,) and bias.dtype in _DTYPES, f"bias must be fp32, bf16 or fp16 [{e}]"
        _same(bias, "bias", dev)
        bias = bias.contiguous()
        b_ptr, b_code = bias.data_ptr(), _DTYPES[bias.dtype]
    if topk_idx is None:
        topk_idx = _empty(t, top_k, dtype=torch.int32, device=logits.device)
    else:
        _out_flat(topk_idx, "topk_idx", (t, top_k), torch.int32, dev)
    if topk_weights is None:
        topk_weights = _empty(t, top_k, dtype=torch.float32, device=logits.device)
    else:
        _out_flat(topk_weights, "topk_weights", (t, top_k), torch.float32, dev)
    _call("moe_route_topk", dev, logits.data_ptr(), _DTYPES[logits.dtype], _ld(logits), b_ptr,
          b_code, t, e, top_k, _SCORES[score], n_group, topk_group, _GROUP_SCORES[group_score],
          1 if renormalize else 0, routed_scaling_factor, topk_idx.data_ptr(),
          topk_weights.data_ptr())
    return topk_idx, topk_weights


def fp4_scales_shape(rows: int, k: int, fmt: str = "nvfp4") -> Tuple[int, int, int, int, int]:
    """Shape ``[ceil(R/128), ceil(runs/4), 32, 4, 4]`` of a matrix's scales: the
    scale of row ``r`` and run ``b`` (16 or 32 columns) is element
    ``[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]``."""
    assert fmt in _FORMATS, "fmt must be 'mxfp4' or 'nvfp4'"
    per = 4 * _RUN[fmt]
    return (rows + 127) // 128, (k + per - 1) // per, 32, 4, 4


def _check_scale(g: Optional[torch.Tensor], name: str, fmt: str, index: int) -> Optional[int]:
    """Address of a tensor scale, ``None`` without one."""
    if g is None:
        return None
    assert fmt == "nvfp4", f"{name} belongs to nvfp4"
    assert g.dtype == torch.float32 and g.numel() == 1, f"{name} must be one float32"
    _same(g, name, index)
    return g.data_ptr()


def _check_matrix(codes: torch.Tensor, scales: torch.Tensor, fmt: str, name: str) -> Tuple[int, int, int]:
    """(rows, K, device index) of a matrix in 4 bits."""
    assert fmt in _FORMATS, "fmt must be 'mxfp4' or 'nvfp4'"
    assert codes.dim() == 2 and codes.dtype == torch.uint8, f"{name}_codes must be uint8 [rows, K/2]"
    r, k = codes.shape
    k *= 2
    assert k >= 32 and k % 32 == 0, "K must be a multiple of 32"
    shape = fp4_scales_shape(r, k, fmt)
    assert scales.dtype == torch.uint8 and scales.shape == shape, \
        f"{name}_scales must be uint8 {list(shape)} (fp4_scales_shape)"
    assert scales.is_contiguous() and scales.data_ptr() % 16 == 0, \
        f"{name}_scales must be contiguous and 16-byte aligned"
    dev = _gpu(codes, f"{name}_codes")
    _same(scales, f"{name}_scales", dev)
    return r, k, dev


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
    assert fmt in _FORMATS, "fmt must be 'mxfp4' or 'nvfp4'"
    assert x.dim() == 2 and x.dtype in _DTYPES, "x must be fp32, bf16 or fp16 [R, K]"
    r, k = x.shape
    assert k >= 32 and k % 32 == 0, "K must be a multiple of 32"
    dev = _gpu(x, "x")
    g_ptr = _check_scale(global_scale, "global_scale", fmt, dev)
    x = _rows(x)
    if codes is None:
        codes = _empty(r, k // 2, dtype=torch.uint8, device=x.device)
    else:
        _out_flat(codes, "codes", (r, k // 2), torch.uint8, dev)
    shape = fp4_scales_shape(r, k, fmt)
    if scales is None:
        scales = _empty(*shape, dtype=torch.uint8, device=x.device)
    else:
        _out_flat(scales, "scales", shape, torch.uint8, dev)
    _call("moe_fp4_quantize", dev, x.data_ptr(), _DTYPES[x.dtype], _ld(x), r, k, _FORMATS[fmt], g_ptr,
          codes.data_ptr(), scales.data_ptr())
    return codes, scales


def dequantize_fp4(codes: torch.Tensor, scales: torch.Tensor, fmt: str = "nvfp4", *,
                   global_scale: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values ``[R, K]`` of a matrix in microscaled 4 bits, rounded to ``dtype``."""
    r, k, dev = _check_matrix(codes, scales, fmt, "input")
    assert dtype in _DTYPES, "dtype must be fp32, bf16 or fp16"
    g_ptr = _check_scale(global_scale, "global_scale", fmt, dev)
    codes = _rows(codes)
    if out is None:
        out = _empty(r, k, dtype=dtype, device=codes.device)
    else:
        _out_flat(out, "out", (r, k), dtype, dev)
    _call("moe_fp4_dequantize", dev, codes.data_ptr(), _ld(codes), scales.data_ptr(), r, k, _FORMATS[fmt],
          g_ptr, out.data_ptr(), _DTYPES[dtype])
    return out


def _product_out(out: Optional[torch.Tensor], t: int, n: int, dtype: torch.dtype,
                 device: torch.device) -> torch.Tensor:
    assert dtype in _DTYPES, "dtype must be fp32, bf16 or fp16"
    if out is None:
        return _empty(t, n, dtype=dtype, device=device)
    _check_out(out, "out", (t, n), dtype, device.index)
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
    t, k, dev = _check_matrix(a_codes, a_scales, fmt, "a")
    n, kb, dev_b = _check_matrix(b_codes, b_scales, fmt, "b")
    assert k == kb, f"a and b must have the same K, not {k} and {kb}"
    assert dev == dev_b, "a and b must be on one device"
    ga = _check_scale(a_global_scale, "a_global_scale", fmt, dev)
    gb = _check_scale(b_global_scale, "b_global_scale", fmt, dev)
    a_codes, b_codes = _rows(a_codes), _rows(b_codes)
    out = _product_out(out, t, n, dtype, a_codes.device)
    _call("moe_fp4_matmul", dev, a_codes.data_ptr(), _ld(a_codes), a_scales.data_ptr(), ga,
          b_codes.data_ptr(), _ld(b_codes), b_scales.data_ptr(), gb, _FORMATS[fmt], t, n, k,
          out.data_ptr(), _DTYPES[dtype], _ld(out))
    return out


@functools.lru_cache(maxsize=1024)
def _linear_workspace(code: int, t: int, k: int) -> int:
    """Bytes that the product of ``t`` tokens wants."""
    n = ctypes.c_size_t()
    st = _lib.load().moe_fp4_linear_workspace_size(code, t, k, ctypes.byref(n))
    if st:
        _raise(st, "moe_fp4_linear_workspace_size")
    return n.value


def linear_fp4(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor, fmt: str = "nvfp4", *,
               x_global_scale: Optional[torch.Tensor] = None,
               w_global_scale: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [T, K] . W [N, K]^T`` with ``W`` in microscaled 4 bits: quantises ``x``
    (fp32, bf16 or fp16) as ``quantize_fp4`` does and multiplies as
    ``matmul_fp4`` does, in ``dtype`` (default: ``x``'s).  ``out`` must not overlap
    ``x``; other columns of the same rows are fine."""
    n, k, dev = _check_matrix(w_codes, w_scales, fmt, "w")
    assert x.dim() == 2 and x.dtype in _DTYPES, "x must be fp32, bf16 or fp16 [T, K]"
    t = x.shape[0]
    assert x.shape[1] == k, f"x must be [T, {k}]"
    _same(x, "x", dev)
    gx = _check_scale(x_global_scale, "x_global_scale", fmt, dev)
    gw = _check_scale(w_global_scale, "w_global_scale", fmt, dev)
    x, w_codes = _rows(x), _rows(w_codes)
    dtype = x.dtype if dtype is None else dtype
    out = _product_out(out, t, n, dtype, x.device)
    ws, ws_ptr, nbytes = None, None, _linear_workspace(_FORMATS[fmt], t, k)
    if nbytes:
        # codes and scales of x live for this call only: a buffer of the current
        # stream (or of the graph being captured), never shared between calls
        ws = _empty(nbytes, dtype=torch.uint8, device=x.device)
        ws_ptr = ws.data_ptr()
    _call("moe_fp4_linear", dev, x.data_ptr(), _DTYPES[x.dtype], _ld(x), gx, w_codes.data_ptr(),
          _ld(w_codes), w_scales.data_ptr(), gw, _FORMATS[fmt], t, n, k, out.data_ptr(), _DTYPES[dtype],
          _ld(out), ws_ptr, nbytes)
    return out


def fp4_device_error(device: Optional[torch.device] = None) -> Tuple[int, int]:
    """(code, info) of the first device-side wait of a 4-bit product that ran out
    on ``device`` since the last one that was read; (0, 0) if none.  Blocks."""
    code, info = ctypes.c_int32(0), ctypes.c_int32(0)
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream().cuda_stream
        st = _lib.load().moe_fp4_device_error(stream, ctypes.byref(code), ctypes.byref(info))
    if st:
        _raise(st, "moe_fp4_device_error")
    return code.value, info.value
