"""Softmax cross entropy of a linear head, its backward and its autograd form
(``csrc/gdn_xent.hip``).  No counterpart in the reference."""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DTYPE_CODE, _PLANS_MAX, _check_devices, _check_sizes, _first_order, _launch, _needs_grad
from .scan import _failed, _like, _sig

_MAX_STRIDE = 1 << 22

_FWD_PLANS = {}
_BWD_PLANS = {}


def _check_rows(t, name):
    """Rows are read 16 bytes at a time, a tile's rows within 31 bits of its first."""
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous (stride {t.stride(-1)}); "
                         "call .contiguous()")
    if t.data_ptr() % 16 != 0 or (t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) > _MAX_STRIDE)):
        raise ValueError(f"{name}: rows must be 16-byte aligned, at most {_MAX_STRIDE} elements apart (data_ptr and "
                         f"stride {t.stride(0)}); call .contiguous()")


def _flat(t):
    """[..., D] as [N, D] (a copy only where its strides need one)."""
    return t.flatten(0, -2) if isinstance(t, torch.Tensor) and t.dim() > 2 else t


def _validate(x, weight, target):
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        raise ValueError("x must be [..., D]")
    D = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] != D or weight.shape[0] < 1:
        raise ValueError(f"weight must be [V, D] with x's D={D}")
    if x.dtype not in (torch.float16, torch.bfloat16) or weight.dtype != x.dtype:
        raise ValueError(f"x and weight must share float16 or bfloat16 (got {x.dtype}, {weight.dtype})")
    if D < 8 or D % 8 != 0:
        raise ValueError(f"D={D} not supported (a multiple of 8)")
    if not isinstance(target, torch.Tensor) or target.shape != x.shape[:-1] or \
            target.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"target must be an int64 or int32 tensor of {tuple(x.shape[:-1])}")
    if x.device.type != "cuda":
        raise ValueError(f"linear_xent runs on a ROCm GPU (got {x.device}); there is no CPU path")
    _check_devices(x, weight, target)


def _plan(x, weight, target, lse, dloss, backward):
    _validate(x, weight, target)
    if backward:
        for name, t in (("lse", lse), ("dloss", dloss)):
            if not isinstance(t, torch.Tensor) or t.shape != target.shape or t.dtype != torch.float32:
                raise ValueError(f"{name} must be float32 {tuple(target.shape)}")
        _check_devices(x, lse, dloss)
    x2 = _flat(x)
    if x.numel() > 0:
        _check_rows(x2, "x")
    _check_rows(weight, "weight")
    _check_sizes(*x2.shape, weight.shape[0])
    P = _lib.GdnXentParams()
    P.N, P.D, P.V = x2.shape[0], x2.shape[1], weight.shape[0]
    P.x_stride, P.w_stride = x2.stride(0), weight.stride(0)
    P.dtype = _DTYPE_CODE[x.dtype]
    lib = _lib.load_library()
    ws = (lib.gdn_xent_bwd_workspace_size if backward else lib.gdn_xent_workspace_size)(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"linear_xent does not support x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    return bytes(P), int(ws)


def _planned(plans, x, weight, target, lse=None, dloss=None):
    """The plan of a signature seen before, or a new one.  (The alignment is of
    this call's pointers: part of the signature.)"""
    try:
        key = (_sig(x), _sig(weight), _sig(target), _sig(lse), _sig(dloss), (x.data_ptr() | weight.data_ptr()) & 15)
        plan = plans.get(key)
    except (AttributeError, TypeError):     # not tensors: the checks say which
        key, plan = None, None
    if plan is None:
        plan = _plan(x, weight, target, lse, dloss, plans is _BWD_PLANS)
        if key is not None:
            if len(plans) >= _PLANS_MAX:
                plans.clear()
            plans[key] = plan
    return plan


def _targets(target):
    """As the kernels read them: contiguous int64."""
    return target if target.dtype == torch.int64 and target.is_contiguous() else target.to(torch.int64).contiguous()


def _run(x, weight, target):
    params, ws_bytes = _planned(_FWD_PLANS, x, weight, target)
    x2, t = _flat(x), _targets(target)
    loss = torch.empty(target.shape, dtype=torch.float32, device=x.device)
    lse = torch.empty_like(loss)
    if t.numel() > 0:
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
        P = _lib.GdnXentParams.from_buffer_copy(params)
        P.x, P.w, P.target = x2.data_ptr(), weight.data_ptr(), t.data_ptr()
        P.loss, P.lse = loss.data_ptr(), lse.data_ptr()
        P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
        status = _launch(_lib.load_library().gdn_xent_launch, P, x.device)
        if status != 0:
            raise _failed("gdn_xent_launch", status)
    return loss, lse


def linear_xent(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, return_lse: bool = False):
    """Cross entropy of the softmax over the logits ``x @ weight.T``, row by row:

        ``loss = log sum_v e^{logit_v} - logit_target``,

    the logits made in fp32 in pieces of the vocabulary and never kept.

    Args:
      x: ``[..., D]`` float16 or bfloat16, D a multiple of 8, 16-byte aligned
        rows; weight: ``[V, D]``, the same dtype.
      target: ``[...]`` int64 or int32.  A row whose target is outside
        ``[0, V)`` (padding) does not count: its loss and gradients are 0,
        whatever the row holds.
      return_lse: also return ``log sum_v e^{logit_v}`` (0 for rows that do not
        count), as ``linear_xent_bwd`` takes it.

    Returns ``loss [...]`` float32 (a mean over the rows that count is
    ``loss.sum() / counts.sum()``), and with ``return_lse`` ``(loss, lse)``.
    ``loss`` is differentiable in x and weight (``lse`` is not).
    """
    if _needs_grad(x, weight):
        loss, lse = _XentFunction.apply(x, weight, target)
    else:
        loss, lse = _run(x, weight, target)
    return (loss, lse) if return_lse else loss


def _run_bwd(x, weight, target, lse, dloss):
    params, ws_bytes = _planned(_BWD_PLANS, x, weight, target, lse, dloss)
    dx, dw = _like(x), _like(weight)
    if target.numel() == 0:
        return dx, dw.zero_()
    x2, t, l = _flat(x), _targets(target), lse.contiguous()
    # one value for all rows, as a sum or mean hands it over, is read with a stride of 0
    step = 0
    if any(s != 0 for s, n in zip(dloss.stride(), dloss.shape) if n > 1):
        dloss, step = dloss.contiguous(), 1
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    P = _lib.GdnXentParams.from_buffer_copy(params)
    P.x, P.w, P.target = x2.data_ptr(), weight.data_ptr(), t.data_ptr()
    P.lse, P.dloss, P.dloss_stride = l.data_ptr(), dloss.data_ptr(), step
    P.dx, P.dw = dx.data_ptr(), dw.data_ptr()
    P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_xent_bwd_launch, P, x.device)
    if status != 0:
        raise _failed("gdn_xent_bwd_launch", status)
    return dx, dw


def linear_xent_bwd(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, lse: torch.Tensor,
                    dloss: torch.Tensor):
    """Gradients ``(dx, dweight)`` of ``linear_xent`` given ``dloss [...]``
    float32 and the ``lse`` that it returned:

        ``G = dloss (e^{logit - lse} - [v = target])``, ``dx = G weight``, ``dweight = G^T x``.

    The logits are made again, piece by piece of the vocabulary (about 128 MiB
    of G at a time); all sums are fp32 in a fixed order, so repeated calls give
    the same bits."""
    return _run_bwd(x, weight, target, lse, dloss)


class _XentFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target):
        loss, lse = _run(x, weight, target)
        ctx.save_for_backward(x, weight, target, lse)
        ctx.mark_non_differentiable(lse)
        return loss, lse

    @staticmethod
    @_first_order
    def backward(ctx, dloss, _):
        return (*_run_bwd(*ctx.saved_tensors, dloss), None)
