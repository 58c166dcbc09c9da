"""Elementwise gated linear recurrence ``h_t = e^{g_t} h_{t-1} + x_t``, its
backward and its autograd form (``csrc/gdn_scan.hip``).  No counterpart in the
reference."""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .ops import _DTYPE_CODE, _PLANS_MAX, _check_devices, _code, _first_order, _launch, _needs_grad, _offsets

_FWD_PLANS = {}
_BWD_PLANS = {}


def _sig(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _like(t, dtype=None):
    """A new dense tensor of t's shape (empty_like, the cheaper call, keeps the
    order of dense strides)."""
    if t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device)


def _failed(name, status):
    return RuntimeError(f"{name} failed ({status}): {_lib.op_status_string(status)}")


def _validate(x, g, h0, n_seq):
    """Checks shapes, dtypes and devices; returns (B, T, D, N)."""
    for name, t in (("x", x), ("g", g)):
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise ValueError(f"{name} must be a [B, T, D] tensor")
    B, T, D = x.shape
    if tuple(g.shape) != (B, T, D):
        raise ValueError(f"g must be [B, T, D] = ({B}, {T}, {D}), got {tuple(g.shape)}")
    _code(x, "x")
    if g.dtype != x.dtype and g.dtype != torch.float32:
        raise ValueError(f"g must be float32 or x's dtype {x.dtype}, got {g.dtype}")
    if B <= 0 or D <= 0:
        raise ValueError(f"B and D must be positive (got B={B}, D={D})")
    if n_seq is not None and B != 1:
        raise ValueError(f"with cu_seqlens the inputs hold one packed batch: B must be 1, got {B}")
    N = B if n_seq is None else n_seq
    _check_state(h0, "h0", N, D)
    if x.device.type != "cuda":
        raise ValueError(f"gated_scan runs on a ROCm GPU (got {x.device}); there is no CPU path")
    _check_devices(x, g, h0)
    for name, t in (("x", x), ("g", g)):
        _check_columns(t, name)
    return B, T, D, N


def _check_state(t, name, N, D):
    if t is None:
        return
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (N, D) or t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 [N, D] = [{N}, {D}]")
    _check_columns(t, name)


def _check_columns(t, name):
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous (stride {t.stride(-1)}); "
                         "call .contiguous()")


def _params(x, g, h0, B, T, D, N):
    P = _lib.GdnScanParams()
    P.B, P.T, P.D, P.N = B, T, D, N
    P.x_dtype, P.g_dtype = _DTYPE_CODE[x.dtype], _DTYPE_CODE[g.dtype]
    P.x_stride[:] = x.stride()[:2]
    P.g_stride[:] = g.stride()[:2]
    P.h0_stride = h0.stride(0) if h0 is not None else 0
    return P


def _fwd_plan(x, g, h0, n_seq, return_states):
    B, T, D, N = _validate(x, g, h0, n_seq)
    P = _params(x, g, h0, B, T, D, N)
    P.y_stride[:] = (T * D, D)
    lib = _lib.load_library()
    P.cu_seqlens = 1 if n_seq is not None else None     # only whether it is set counts here
    P.states = 1 if return_states else None
    ws = lib.gdn_scan_workspace_size(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"gated_scan does not support B={B} T={T} D={D}")
    slots = lib.gdn_scan_slots(B, T, N, int(n_seq is not None))
    P.cu_seqlens = P.states = None
    return bytes(P), int(ws), (N, D), (slots, D)


def _run(x, g, h0, cu, n_seq, return_states):
    try:
        key = (_sig(x), _sig(g), _sig(h0), n_seq, return_states)
        plan = _FWD_PLANS.get(key)
    except (AttributeError, TypeError):     # not tensors: _validate says which
        key, plan = None, None
    if plan is None:
        plan = _fwd_plan(x, g, h0, n_seq, return_states)
        if key is not None:
            if len(_FWD_PLANS) >= _PLANS_MAX:
                _FWD_PLANS.clear()
            _FWD_PLANS[key] = plan
    params, ws_bytes, shape_fs, shape_st = plan
    dev = x.device
    y = _like(x)
    fs = _like(h0) if h0 is not None else x.new_empty(shape_fs, dtype=torch.float32)
    states = x.new_empty(shape_st, dtype=torch.float32) if return_states else None
    ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes > 0 else None
    P = _lib.GdnScanParams.from_buffer_copy(params)
    P.x, P.g = x.data_ptr(), g.data_ptr()
    P.h0 = h0.data_ptr() if h0 is not None else None
    P.y, P.final_state = y.data_ptr(), fs.data_ptr()
    P.states = states.data_ptr() if states is not None else None
    P.cu_seqlens = cu.data_ptr() if cu is not None else None
    if ws is not None:
        P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_scan_launch, P, dev)
    if status != 0:
        raise _failed("gdn_scan_launch", status)
    return y, fs, states


def _seqs(x, cu_seqlens):
    if cu_seqlens is None:
        return None, None
    if not isinstance(x, torch.Tensor):
        raise ValueError("x must be a [B, T, D] tensor")
    return _offsets(cu_seqlens, x.device)


def gated_scan(x: torch.Tensor, g: torch.Tensor, h0: Optional[torch.Tensor] = None, *,
               cu_seqlens: Optional[torch.Tensor] = None, return_states: bool = False):
    """Elementwise gated linear recurrence ``h_t = e^{g_t} h_{t-1} + x_t``,
    ``y_t = h_t``, the state in fp32.

    Args:
      x: ``[B, T, D]`` float16, bfloat16 or float32, last dim contiguous; any
        T and D.
      g: ``[B, T, D]`` log-decay gates, float32 or x's dtype (``-inf`` forgets
        the state).
      h0: optional ``[N, D]`` float32 initial state (N = B without
        ``cu_seqlens``).
      cu_seqlens: optional int64 ``[N + 1]`` row offsets of N sequences packed
        along t (B = 1), rising from 0 to T.  They are not read on the host
        (the call does not wait for the device); the kernels clamp them to
        ``[0, T]``, and rows outside every sequence are left unwritten.
      return_states: also return the states at the chunks' starts, which
        ``gated_scan_bwd`` takes instead of computing them again.

    Returns:
      ``y [B, T, D]`` in x's dtype and ``final_state [N, D]`` float32, and
      with ``return_states`` the states.  ``y`` and ``final_state`` are
      differentiable when an input requires grad.
    """
    cu, n_seq = _seqs(x, cu_seqlens)
    if _needs_grad(x, g, h0):
        y, fs, states = _ScanFunction.apply(x, g, h0, cu, n_seq)
    else:
        y, fs, states = _run(x, g, h0, cu, n_seq, return_states)
    return (y, fs, states) if return_states else (y, fs)


def _bwd_plan(x, g, h0, dy, dfinal, states, n_seq, need_dh0):
    B, T, D, N = _validate(x, g, h0, n_seq)
    if not isinstance(dy, torch.Tensor) or dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must have x's shape {tuple(x.shape)} and dtype {x.dtype}")
    _check_columns(dy, "dy")
    _check_state(dfinal, "dfinal", N, D)
    if states is not None and not isinstance(states, torch.Tensor):
        raise ValueError("states must be the tensor that gated_scan returned")
    _check_devices(x, dy, dfinal, states)
    P = _params(x, g, h0, B, T, D, N)
    P.dy_stride[:] = dy.stride()[:2]
    P.dx_stride[:] = P.dg_stride[:] = (T * D, D)
    P.dfinal_stride = dfinal.stride(0) if dfinal is not None else 0
    lib = _lib.load_library()
    slots = lib.gdn_scan_slots(B, T, N, int(n_seq is not None))
    if states is not None:
        if tuple(states.shape) != (slots, D) or states.dtype != torch.float32 or not states.is_contiguous():
            raise ValueError(f"states must be the float32 [{slots}, {D}] tensor that gated_scan returned")
    P.cu_seqlens = 1 if n_seq is not None else None
    P.states = 1 if states is not None else None
    ws = lib.gdn_scan_bwd_workspace_size(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"gated_scan_bwd does not support B={B} T={T} D={D}")
    P.cu_seqlens = P.states = None
    return bytes(P), int(ws), (N, D) if need_dh0 else None


def _run_bwd(x, g, h0, dy, dfinal, states, cu, n_seq, need_dh0):
    # autograd may hand over any layout, e.g. the expansion of a scalar
    if isinstance(dy, torch.Tensor) and dy.dim() == 3 and dy.stride(-1) != 1:
        dy = dy.contiguous()
    if isinstance(dfinal, torch.Tensor) and dfinal.dim() == 2 and dfinal.stride(-1) != 1:
        dfinal = dfinal.contiguous()
    try:
        key = (_sig(x), _sig(g), _sig(h0), _sig(dy), _sig(dfinal), _sig(states), n_seq, need_dh0)
        plan = _BWD_PLANS.get(key)
    except (AttributeError, TypeError):
        key, plan = None, None
    if plan is None:
        plan = _bwd_plan(x, g, h0, dy, dfinal, states, n_seq, need_dh0)
        if key is not None:
            if len(_BWD_PLANS) >= _PLANS_MAX:
                _BWD_PLANS.clear()
            _BWD_PLANS[key] = plan
    params, ws_bytes, shape_dh0 = plan
    dev = x.device
    dx, dg = _like(x), _like(g)
    dh0 = x.new_empty(shape_dh0, dtype=torch.float32) if shape_dh0 is not None else None
    ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes > 0 else None
    P = _lib.GdnScanParams.from_buffer_copy(params)
    P.x, P.g, P.dy = x.data_ptr(), g.data_ptr(), dy.data_ptr()
    P.h0 = h0.data_ptr() if h0 is not None else None
    P.dfinal = dfinal.data_ptr() if dfinal is not None else None
    P.dx, P.dg = dx.data_ptr(), dg.data_ptr()
    P.dh0 = dh0.data_ptr() if dh0 is not None else None
    P.states = states.data_ptr() if states is not None else None
    P.cu_seqlens = cu.data_ptr() if cu is not None else None
    if ws is not None:
        P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_scan_bwd_launch, P, dev)
    if status != 0:
        raise _failed("gdn_scan_bwd_launch", status)
    return dx, dg, dh0


def gated_scan_bwd(x: torch.Tensor, g: torch.Tensor, h0: Optional[torch.Tensor], dy: torch.Tensor,
                   dfinal: Optional[torch.Tensor] = None, *, cu_seqlens: Optional[torch.Tensor] = None,
                   states: Optional[torch.Tensor] = None, need_dh0: bool = True):
    """Gradients of ``gated_scan`` given ``dy`` (of ``y``, x's shape and dtype)
    and ``dfinal`` (of ``final_state``, float32 ``[N, D]``, or None for zero):

        ``dh_t = dy_t + e^{g_{t+1}} dh_{t+1}``, ``dx = dh``,
        ``dg_t = dh_t e^{g_t} h_{t-1}``, ``dh0 = e^{g_1} dh_1``.

    Returns ``(dx, dg, dh0)`` in the inputs' dtypes (``dh0`` float32, None
    unless ``need_dh0``).  ``states``: what ``gated_scan(..., return_states=
    True)`` returned for the same inputs; without it the states are computed
    again from x, g and h0.  Packed sequences as in ``gated_scan``.
    """
    cu, n_seq = _seqs(x, cu_seqlens)
    return _run_bwd(x, g, h0, dy, dfinal, states, cu, n_seq, need_dh0)


class _ScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, h0, cu, n_seq):
        y, fs, states = _run(x, g, h0, cu, n_seq, True)
        ctx.save_for_backward(x, g, h0, cu, states)
        ctx.mark_non_differentiable(states)
        ctx.set_materialize_grads(False)
        return y, fs, states

    @staticmethod
    @_first_order
    def backward(ctx, dy, dfs, _):
        x, g, h0, cu, states = ctx.saved_tensors
        n_seq = None
        if cu is not None:
            cu, n_seq = _offsets(cu, x.device)      # saved-tensor hooks may hand back another
        if dy is None:
            dy = torch.zeros_like(x)
        need_dh0 = h0 is not None and ctx.needs_input_grad[2]
        dx, dg, dh0 = _run_bwd(x, g, h0, dy, dfs, states, cu, n_seq, need_dh0)
        return dx, dg, dh0, None, None
