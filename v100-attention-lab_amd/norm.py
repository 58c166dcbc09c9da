"""Root-mean-square norm with the residual's addition, its backward and its
8-bit form (``csrc/gdn_norm.hip``).  No counterpart in the reference."""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .ops import _DTYPE_CODE, _PLANS_MAX, _check_devices, _code, _first_order, _launch, _needs_grad
from .scan import _check_columns, _failed, _like, _sig

_FWD_PLANS = {}
_BWD_PLANS = {}


def _rows(t):
    """(outer, inner, strides) of t's rows: the leading dimensions, at most two."""
    if t.dim() == 1:
        return 1, 1, (0, 0)
    if t.dim() == 2:
        return 1, t.shape[0], (0, t.stride(0))
    return t.shape[0], t.shape[1], t.stride()[:2]


def _at_most_3d(t):
    """t with its leading dimensions but the last joined (a copy only where its
    strides need one)."""
    return t.flatten(0, -3) if isinstance(t, torch.Tensor) and t.dim() > 3 else t


def _check_x(x, name, weight):
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must be a [..., D] tensor")
    _code(x, name)
    D = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or tuple(weight.shape) != (D,):
        raise ValueError(f"weight must be [D] = [{D}]")
    if x.device.type != "cuda":
        raise ValueError(f"add_rms_norm runs on a ROCm GPU (got {x.device}); there is no CPU path")
    _check_columns(x, name)
    _check_columns(weight, "weight")


def _check_like(t, name, shape, dtypes):
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dict.fromkeys(dtypes))}, got {t.dtype}")
    _check_columns(t, name)


def _dense(outer, inner, D):
    return (inner * D, D)


def _fwd_plan(x, weight, residual, eps, fp8, group):
    _check_x(x, "x", weight)
    _check_like(weight, "weight", weight.shape, (x.dtype, torch.float32))
    if residual is not None:
        _check_like(residual, "residual", x.shape, (x.dtype, torch.float32))
    _check_devices(x, weight, residual)
    D = x.shape[-1]
    if group is not None and (group != 128 or D % 128 != 0):
        raise ValueError(f"group must be None or 128 dividing D={D}, got {group}")
    P = _lib.GdnNormParams()
    P.n_outer, P.n_inner, strides = _rows(x)
    P.x_stride[:] = strides
    if residual is not None:
        P.res_stride[:] = _rows(residual)[2]
    P.y_stride[:] = P.r_out_stride[:] = _dense(P.n_outer, P.n_inner, D)
    P.D, P.eps, P.group = D, float(eps), group or 0
    P.x_dtype, P.w_dtype = _DTYPE_CODE[x.dtype], _DTYPE_CODE[weight.dtype]
    P.r_dtype = _DTYPE_CODE[x.dtype if residual is None else residual.dtype]
    return bytes(P), (*x.shape[:-1], D // (group or D))


def _run(x, weight, residual, eps, fp8, group):
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x3, residual3 = _at_most_3d(x), _at_most_3d(residual)
    try:
        key = (_sig(x3), _sig(weight), _sig(residual3), float(eps), fp8, group, shape)
        plan = _FWD_PLANS.get(key)
    except (AttributeError, TypeError):     # not tensors: the checks say which
        key, plan = None, None
    if plan is None:
        if residual is not None and getattr(residual, "shape", None) != shape:
            raise ValueError(f"residual must have shape {shape and tuple(shape)}")
        plan = _fwd_plan(x3, weight, residual3, eps, fp8, group)
        if x3 is not x:
            plan = plan[0], (*shape[:-1], shape[-1] // (group or shape[-1]))
        if key is not None:
            if len(_FWD_PLANS) >= _PLANS_MAX:
                _FWD_PLANS.clear()
            _FWD_PLANS[key] = plan
    params, shape_scale = plan
    dev = x.device
    y = _like(x, torch.float8_e4m3fn if fp8 else None)
    scale = x.new_empty(shape_scale, dtype=torch.float32) if fp8 else None
    P = _lib.GdnNormParams.from_buffer_copy(params)
    P.x, P.w, P.y = x3.data_ptr(), weight.data_ptr(), y.data_ptr()
    r = x
    if residual is not None:
        r = _like(residual)
        P.res, P.r_out = residual3.data_ptr(), r.data_ptr()
    if fp8:
        P.scale = scale.data_ptr()
    if y.numel() > 0:
        status = _launch(_lib.load_library().gdn_norm_launch, P, dev)
        if status != 0:
            raise _failed("gdn_norm_launch", status)
    return y, scale, r


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 eps: float = 1e-6):
    """``r = x + residual``, ``y = r / sqrt(mean(r^2) + eps) * weight`` over the
    last dim, in one launch, the sums in fp32.

    Args:
      x: ``[..., D]`` float16, bfloat16 or float32, last dim contiguous.
      weight: ``[D]`` float32 or x's dtype.
      residual: optional, x's shape, float32 or x's dtype.

    Returns:
      ``y`` in x's dtype and ``r`` in the residual's (x itself without one).
      ``y`` is formed from the fp32 sum, before r is rounded to its dtype; the
      gradient is taken at the stored r.  Both are differentiable when an
      input requires grad.
    """
    if _needs_grad(x, weight, residual):
        eps = float(eps)        # (kept for the backward)
        if residual is None:
            return _NormFunction.apply(x, weight, None, eps), x
        return _NormFunction.apply(x, weight, residual, eps)
    y, _, r = _run(x, weight, residual, eps, False, None)
    return y, r


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                     eps: float = 1e-6, *, group: Optional[int] = None):
    """``add_rms_norm`` with an 8-bit output for the product that follows.

    Returns ``(y, scale, r)``: ``y`` float8_e4m3fn, ``scale`` float32 with
    ``y * scale`` the norm's output; scale is ``max|.| / 448`` over each row
    (``[..., 1]``) or, with ``group=128``, over each 128 columns
    (``[..., D / 128]``).  A group of zeros has scale 0.  Not differentiable.
    """
    if _needs_grad(x, weight, residual):
        raise NotImplementedError("add_rms_norm_fp8 has no gradient: use add_rms_norm in training")
    return _run(x, weight, residual, eps, True, group)


def _bwd_plan(r, weight, dy, dr, eps, x_dtype):
    _check_x(r, "r", weight)
    _check_like(dy, "dy", r.shape, (x_dtype,))
    if r.dtype not in (x_dtype, torch.float32):
        raise ValueError(f"r must be {x_dtype} (dy's dtype) or float32, got {r.dtype}")
    _check_like(weight, "weight", weight.shape, (x_dtype, torch.float32))
    if dr is not None:
        _check_like(dr, "dr", r.shape, (r.dtype,))
    _check_devices(r, weight, dy, dr)
    D = r.shape[-1]
    P = _lib.GdnNormParams()
    P.n_outer, P.n_inner, strides = _rows(r)
    P.r_stride[:] = strides
    P.dy_stride[:] = _rows(dy)[2]
    if dr is not None:
        P.dr_in_stride[:] = _rows(dr)[2]
    P.dr_stride[:] = P.dx_stride[:] = _dense(P.n_outer, P.n_inner, D)
    P.D, P.eps = D, float(eps)
    P.x_dtype, P.r_dtype, P.w_dtype = _DTYPE_CODE[x_dtype], _DTYPE_CODE[r.dtype], _DTYPE_CODE[weight.dtype]
    ws = _lib.load_library().gdn_norm_bwd_workspace_size(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"add_rms_norm_bwd does not support rows of shape {tuple(r.shape)}")
    return bytes(P), int(ws)


def _run_bwd(r, weight, dy, dr, eps, need_dx):
    # autograd may hand over any layout, e.g. the expansion of a scalar
    dy, dr = (t.contiguous() if isinstance(t, torch.Tensor) and t.dim() > 0 and t.stride(-1) != 1 else t
              for t in (dy, dr))
    r3, dy3, dr3 = _at_most_3d(r), _at_most_3d(dy), _at_most_3d(dr)
    try:
        key = (_sig(r3), _sig(weight), _sig(dy3), _sig(dr3), float(eps))
        plan = _BWD_PLANS.get(key)
    except (AttributeError, TypeError):
        key, plan = None, None
    if plan is None:
        for name, t in (("r", r), ("dy", dy)):
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a [..., D] tensor")
        plan = _bwd_plan(r3, weight, dy3, dr3, eps, dy.dtype)
        if key is not None:
            if len(_BWD_PLANS) >= _PLANS_MAX:
                _BWD_PLANS.clear()
            _BWD_PLANS[key] = plan
    params, ws_bytes = plan
    dev = r.device
    out = _like(r)
    dx = _like(dy) if need_dx else None
    dw = _like(weight)
    ws = r.new_empty(ws_bytes, dtype=torch.uint8)
    P = _lib.GdnNormParams.from_buffer_copy(params)
    P.r, P.w, P.dy = r3.data_ptr(), weight.data_ptr(), dy3.data_ptr()
    P.dr_in = dr3.data_ptr() if dr is not None else None
    P.dr, P.dw = out.data_ptr(), dw.data_ptr()
    P.dx = dx.data_ptr() if dx is not None else None
    P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_norm_bwd_launch, P, dev)
    if status != 0:
        raise _failed("gdn_norm_bwd_launch", status)
    return out, dx, dw


def add_rms_norm_bwd(r: torch.Tensor, weight: torch.Tensor, dy: torch.Tensor,
                     dr: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """Gradients of ``add_rms_norm`` at its output ``r``, given ``dy`` (of y) and
    ``dr`` (of r, or None for zero):

        ``n = r / sqrt(mean(r^2) + eps)``,
        ``dr + (weight dy - n mean(weight dy n)) / sqrt(mean(r^2) + eps)``,
        ``dweight = sum over rows of dy n``.

    Returns ``(dr, dweight)``: the first, in r's dtype, is the gradient of
    both x and the residual.
    """
    out, _, dw = _run_bwd(r, weight, dy, dr, eps, False)
    return out, dw


class _NormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, r = _run(x, weight, residual, eps, False, None)
        ctx.save_for_backward(r, weight)
        ctx.eps, ctx.has_res, ctx.x_dtype = eps, residual is not None, x.dtype
        ctx.set_materialize_grads(False)
        return (y, r) if residual is not None else y

    @staticmethod
    @_first_order
    def backward(ctx, dy, dr=None):
        r, weight = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros(r.shape, dtype=ctx.x_dtype, device=r.device)
        out, dx, dw = _run_bwd(r, weight, dy, dr, ctx.eps, ctx.x_dtype != r.dtype)
        return (out if dx is None else dx), dw, (out if ctx.has_res else None), None
