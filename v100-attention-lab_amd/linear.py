"""Products in e4m3 with scales along the contraction, and the quantisers of
their operands (``csrc/gdn_fp8_linear.hip``).  No counterpart in the reference."""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .ops import _DTYPE_CODE, _PLANS_MAX, _check_devices, _check_sizes, _code, _launch, _needs_grad
from .scan import _failed, _like, _sig

FP8 = torch.float8_e4m3fn
BLOCK = 128
_MAX_STRIDE = 1 << 23

_PLANS = {}
_QUANT_PLANS = {}


def _flat(t):
    """[..., D] as [N, D] (a copy only where its strides need one)."""
    return t.flatten(0, -2) if t.dim() > 2 else t if t.dim() == 2 else t[None]


def _check_rows(t, name):
    """Rows are read 16 bytes at a time (t: [N, D])."""
    if t.numel() == 0:
        return
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous (stride {t.stride(-1)}); "
                         "call .contiguous()")
    if t.data_ptr() % 16 != 0 or (t.shape[0] > 1 and t.stride(0) * t.element_size() % 16):
        raise ValueError(f"{name}: rows must be 16-byte aligned (data_ptr and stride {t.stride(0)}); call .contiguous()")


def _quant_plan(x, mode, name):
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be [..., D]")
    _code(x, "x")
    D = x.shape[-1]
    if D < BLOCK or D % BLOCK != 0:
        raise ValueError(f"D={D} not supported (a multiple of {BLOCK})")
    if x.device.type != "cuda":
        raise ValueError(f"{name} runs on a ROCm GPU (got {x.device}); there is no CPU path")
    x2 = _flat(x)
    _check_rows(x2, "x")
    lead = tuple(x.shape[:-1])
    scale = {_lib.FP8_ROWS: (*lead, 1), _lib.FP8_GROUPS: (*lead, D // BLOCK)}.get(mode)
    if scale is None:
        scale = (-(-lead[0] // BLOCK), D // BLOCK)
    _check_sizes(*x2.shape)
    P = _lib.GdnFp8QuantParams()
    P.x_stride, P.rows, P.D = x2.stride(0), x2.shape[0], D
    P.x_dtype, P.mode = _DTYPE_CODE[x.dtype], mode
    return bytes(P), scale, x.dim() == 2


def _quantize(x, mode, name):
    if _needs_grad(x):
        raise NotImplementedError(f"{name} has no gradient")
    try:
        key = (_sig(x), mode, x.data_ptr() & 15)
        plan = _QUANT_PLANS.get(key)
    except (AttributeError, TypeError):     # not a tensor: _quant_plan says so
        key, plan = None, None
    if plan is None:
        plan = _quant_plan(x, mode, name)
        if key is not None:
            if len(_QUANT_PLANS) >= _PLANS_MAX:
                _QUANT_PLANS.clear()
            _QUANT_PLANS[key] = plan
    params, shape, rows = plan
    q = _like(x, FP8)
    scale = x.new_empty(shape, dtype=torch.float32)
    if q.numel() > 0:
        x2 = x if rows else _flat(x)
        P = _lib.GdnFp8QuantParams.from_buffer_copy(params)
        P.x, P.q, P.scale = x2.data_ptr(), q.data_ptr(), scale.data_ptr()
        status = _launch(_lib.load_library().gdn_fp8_quant_launch, P, x.device)
        if status != 0:
            raise _failed("gdn_fp8_quant_launch", status)
    return q, scale


def quantize_fp8(x: torch.Tensor, *, group: Optional[int] = BLOCK):
    """``x [..., D]`` (float16, bfloat16 or float32, D a multiple of 128, rows
    16-byte aligned) as e4m3 with scales, for ``fp8_linear``.

    Returns ``(q, scale)``: ``q`` float8_e4m3fn, ``scale`` float32 with
    ``q * scale ~ x``; scale is ``max|x| / 448`` over each 128 columns
    (``[..., D / 128]``) or, with ``group=None``, over each row (``[..., 1]``).
    A group of zeros has scale 0.  ``add_rms_norm_fp8`` gives the same of the
    norm's output.
    """
    if group not in (None, BLOCK):
        raise ValueError(f"group must be None or {BLOCK}, got {group}")
    return _quantize(x, _lib.FP8_ROWS if group is None else _lib.FP8_GROUPS, "quantize_fp8")


def quantize_fp8_weight(weight: torch.Tensor):
    """``weight [N, K]`` (as ``torch.nn.Linear`` has it, K a multiple of 128) as
    e4m3 with a scale for each block of 128 x 128: ``(q [N, K], scale
    [ceil(N / 128), K / 128])``."""
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be [N, K]")
    return _quantize(weight, _lib.FP8_BLOCKS, "quantize_fp8_weight")


def _plan(x, x_scale, weight, weight_scale, out_dtype):
    for name, t in (("x", x), ("weight", weight)):
        if not isinstance(t, torch.Tensor) or t.dtype != FP8 or t.dim() < 1:
            raise ValueError(f"{name} must be a float8_e4m3fn tensor, x [..., K] and weight [N, K]")
    lead, K = tuple(x.shape[:-1]), x.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != K or weight.shape[0] < 1:
        raise ValueError(f"weight must be [N, K] with x's K={K}, got {tuple(weight.shape)}")
    if K < BLOCK or K % BLOCK != 0:
        raise ValueError(f"K={K} not supported (a multiple of {BLOCK})")
    N = weight.shape[0]
    if not isinstance(x_scale, torch.Tensor) or x_scale.dtype != torch.float32 or \
            tuple(x_scale.shape) not in ((*lead, K // BLOCK), (*lead, 1)):
        raise ValueError(f"x_scale must be float32 {(*lead, K // BLOCK)} or {(*lead, 1)}")
    blocks = (-(-N // BLOCK), K // BLOCK)
    if not isinstance(weight_scale, torch.Tensor) or weight_scale.dtype != torch.float32 or \
            tuple(weight_scale.shape) != blocks:
        raise ValueError(f"weight_scale must be float32 {blocks}")
    if out_dtype not in _DTYPE_CODE:
        raise ValueError(f"out_dtype {out_dtype} not supported (float32, float16, bfloat16)")
    if x.device.type != "cuda":
        raise ValueError(f"fp8_linear runs on a ROCm GPU (got {x.device}); there is no CPU path")
    _check_devices(x, x_scale, weight, weight_scale)
    x2 = _flat(x)
    for name, t in (("x", x2), ("weight", weight)):
        _check_rows(t, name)
        if t.shape[0] > 1 and t.stride(0) > _MAX_STRIDE:
            raise ValueError(f"{name}: rows may be at most {_MAX_STRIDE} elements apart (stride {t.stride(0)})")
    _check_sizes(*x2.shape, N)
    P = _lib.GdnFp8LinearParams()
    P.M, P.N, P.K = x2.shape[0], N, K
    P.x_stride, P.w_stride = x2.stride(0), weight.stride(0)
    P.group = BLOCK if x_scale.shape[-1] == K // BLOCK else 0
    P.y_dtype = _DTYPE_CODE[out_dtype]
    return bytes(P), (*lead, N), x.dim() == 2, x_scale.is_contiguous() and weight_scale.is_contiguous()


def fp8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(x * x_scale) @ (weight * weight_scale).T`` of e4m3 operands.

    Args:
      x: ``[..., K]`` float8_e4m3fn, K a multiple of 128, 16-byte aligned rows;
        x_scale: float32 ``[..., K / 128]``, of each 128 columns, or ``[..., 1]``
        (as ``quantize_fp8`` and ``add_rms_norm_fp8`` give them).
      weight: ``[N, K]`` float8_e4m3fn; weight_scale: float32
        ``[ceil(N / 128), K / 128]`` (as ``quantize_fp8_weight`` gives them).
      out_dtype: float32 comes from fp32 sums.  float16 and bfloat16 come from
        the 8-bit matrix unit, at more than twice the rate, which cuts each
        product at 2^-13 of the largest of its group of 8: off by up to 2^-10 of
        the sum of the terms' sizes beside the one rounding (about 1.4e-5 of the
        result where the terms are normally distributed; more than its rounding
        where they cancel).

    Returns ``y [..., N]``.  Not differentiable.
    """
    if _needs_grad(x, x_scale, weight, weight_scale):
        raise NotImplementedError("fp8_linear has no gradient: multiply in 16 bits in training")
    try:
        key = (x.shape, x.stride(), x.dtype, x.device, _sig(x_scale), _sig(weight), _sig(weight_scale), out_dtype,
               (x.data_ptr() | weight.data_ptr()) & 15)
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):     # not tensors: _plan says which
        key, plan = None, None
    if plan is None:
        plan = _plan(x, x_scale, weight, weight_scale, out_dtype)
        if key is not None:
            if len(_PLANS) >= _PLANS_MAX:
                _PLANS.clear()
            _PLANS[key] = plan
    params, shape, rows, dense = plan
    x2 = x if rows else _flat(x)
    if not dense:
        x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    y = x.new_empty(shape, dtype=out_dtype)
    if y.numel() > 0:
        P = _lib.GdnFp8LinearParams.from_buffer_copy(params)
        P.x, P.x_scale, P.w, P.w_scale = x2.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr()
        P.y = y.data_ptr()
        status = _launch(_lib.load_library().gdn_fp8_linear_launch, P, x.device)
        if status != 0:
            raise _failed("gdn_fp8_linear_launch", status)
    return y
