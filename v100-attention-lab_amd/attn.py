"""Softmax attention with a sliding window and first keys that stay visible:
prefill, its backward and autograd form, and the newest tokens over a cache
(``csrc/gdn_attn_*.hip``).  No counterpart in the reference."""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .ops import _DTYPE_CODE, _PLANS_MAX, _check_devices, _first_order, _launch, _needs_grad, _offsets
from .scan import _failed, _like, _sig

SUPPORTED_D = (64, 128)
MAX_DECODE_T = 16
_INT_MAX = 2 ** 31 - 1

_FWD_PLANS = {}
_BWD_PLANS = {}
_DECODE_PLANS = {}


def _check_window(window, sinks):
    if window is None:
        window = _INT_MAX
    if not isinstance(window, int) or not isinstance(sinks, int) or window < 1 or sinks < 0:
        raise ValueError(f"window must be a positive int or None and sinks an int >= 0 (got {window}, {sinks})")
    return min(window, _INT_MAX), min(sinks, _INT_MAX)


def _number(scale):
    """scale as a float (or None): plans and the backward keep its value, not a
    tensor that may change."""
    if _needs_grad(scale):
        raise NotImplementedError("scale has no gradient: multiply q by it instead")
    return None if scale is None else float(scale)


def _check_rows(t, name):
    """Rows are read 16 bytes at a time; strides of single indexes do not count."""
    if t.numel() == 0:
        return
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous (stride {t.stride(-1)}); "
                         "call .contiguous()")
    if t.data_ptr() % 16 != 0 or any(s % 8 for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1):
        raise ValueError(f"{name}: rows must be 16-byte aligned (data_ptr and strides {t.stride()[:3]}); "
                         "call .contiguous()")


def _validate(q, k, v, names=("q", "k", "v")):
    for name, t in zip(names, (q, k, v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{names[0]} must be [B, T, Hq, D], {names[1]} and {names[2]} [B, S, Hk, D]")
    B, T, Hq, D = q.shape
    S, Hk = k.shape[1:3]
    if tuple(k.shape) != (B, S, Hk, D) or v.shape != k.shape:
        raise ValueError(f"{names[1]} {tuple(k.shape)} and {names[2]} {tuple(v.shape)} must be "
                         f"[B, S, Hk, D] with {names[0]}'s B={B} and D={D}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{', '.join(names)} must share float16 or bfloat16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    if D not in SUPPORTED_D:
        raise ValueError(f"D={D} not supported (D in {SUPPORTED_D})")
    if B <= 0 or Hk <= 0 or Hq <= 0 or Hq % Hk != 0:
        raise ValueError(f"Hq={Hq} must be a positive multiple of Hk={Hk}, and B={B} positive")
    if q.device.type != "cuda":
        raise ValueError(f"window_attn runs on a ROCm GPU (got {q.device}); there is no CPU path")
    _check_devices(q, k, v)
    for name, t in zip(names, (q, k, v)):
        _check_rows(t, name)
    return B, T, S, Hq, Hk, D


def _aligned(*ts):
    """Whether every pointer is 16-byte aligned (checked by every call: plans
    hold all else)."""
    bits = 0
    for t in ts:
        bits |= t.data_ptr()
    return bits & 15 == 0


def _params(q, k, v, B, T, S, Hq, Hk, D, n_seq, window, sinks, scale):
    if n_seq is not None:
        if B != 1:
            raise ValueError(f"with cu_seqlens the inputs hold one packed batch: B must be 1, got {B}")
        if S != T:
            raise ValueError(f"with cu_seqlens q and k must have the same rows, got {T} and {S}")
    P = _lib.GdnAttnParams()
    P.B, P.Tq, P.Tk, P.N = B, T, S, B if n_seq is None else n_seq
    P.Hq, P.Hk, P.D = Hq, Hk, D
    P.window, P.sinks = window, sinks
    P.scale = D ** -0.5 if scale is None else scale
    P.dtype = _DTYPE_CODE[q.dtype]
    P.q_stride[:], P.k_stride[:], P.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    P.o_stride[:] = (T * Hq * D, Hq * D, D)
    return P


def _seqs(q, cu_seqlens):
    if cu_seqlens is None:
        return None, None
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be [B, T, Hq, D]")
    return _offsets(cu_seqlens, q.device)


def _run(q, k, v, window, sinks, scale, cu, n_seq, need_lse):
    try:
        key = (_sig(q), _sig(k), _sig(v), window, sinks, scale, n_seq)
        plan = _FWD_PLANS.get(key)
    except (AttributeError, TypeError):     # not tensors: _validate says which
        key, plan = None, None
    if plan is None:
        w, s = _check_window(window, sinks)
        dims = _validate(q, k, v)
        P = _params(q, k, v, *dims, n_seq, w, s, scale)
        P.cu_seqlens = 1 if n_seq is not None else None     # only whether it is set counts here
        ws_bytes = _lib.load_library().gdn_attn_workspace_size(ctypes.byref(P))
        if ws_bytes < 0:
            raise ValueError(f"window_attn does not support q {tuple(q.shape)}, k {tuple(k.shape)}")
        P.cu_seqlens = None
        plan = bytes(P), int(ws_bytes)
        if key is not None:
            if len(_FWD_PLANS) >= _PLANS_MAX:
                _FWD_PLANS.clear()
            _FWD_PLANS[key] = plan
    elif not _aligned(q, k, v):
        _validate(q, k, v)
    o = _like(q)
    lse = q.new_empty(q.shape[:3], dtype=torch.float32) if need_lse else None
    params, ws_bytes = plan
    ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes > 0 else None
    P = _lib.GdnAttnParams.from_buffer_copy(params)
    if ws is not None:
        P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    P.q, P.k, P.v, P.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()
    P.lse = lse.data_ptr() if lse is not None else None
    P.cu_seqlens = cu.data_ptr() if cu is not None else None
    status = _launch(_lib.load_library().gdn_attn_launch, P, q.device)
    if status != 0:
        raise _failed("gdn_attn_launch", status)
    return o, lse


def window_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None,
                sinks: int = 0, scale: Optional[float] = None, *,
                cu_seqlens: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal softmax attention with a sliding window and sinks.

    The query rows are the last T positions of a sequence of S keys: row i
    stands at ``p = S - T + i`` and sees key j where ``j <= p`` and
    (``j > p - window`` or ``j < sinks``).  A row that sees no key gives zero.

    Args:
      q: ``[B, T, Hq, D]``; k, v: ``[B, S, Hk, D]``, Hq a multiple of Hk (head
        h reads key head ``h // (Hq // Hk)``); float16 or bfloat16, D in
        {64, 128}, 16-byte aligned rows, any other strides.
      window: keys in reach, the row's own among them; None: all earlier ones.
      sinks: first keys that every later row sees.
      scale: of the scores, a number, default ``D ** -0.5``.
      cu_seqlens: optional int64 ``[N + 1]`` offsets of N sequences packed
        along t (B = 1, S = T), rising from 0 to T.  They are not read on the
        host; the kernels clamp them to ``[0, T]``, and rows outside every
        sequence are left unwritten.
      return_lse: also return ``log sum e^{score}`` over the visible keys,
        ``[B, T, Hq]`` float32 (-inf for a row without any).

    Returns ``o [B, T, Hq, D]``, and with ``return_lse`` ``(o, lse)``.  ``o``
    is differentiable (``lse`` is not).
    """
    cu, n_seq = _seqs(q, cu_seqlens)
    scale = _number(scale)
    if _needs_grad(q, k, v):
        o, lse = _AttnFunction.apply(q, k, v, window, sinks, scale, cu, n_seq)
    else:
        o, lse = _run(q, k, v, window, sinks, scale, cu, n_seq, return_lse)
    return (o, lse) if return_lse else o


def _bwd_plan(q, k, v, o, lse, do, window, sinks, scale, n_seq):
    w, s = _check_window(window, sinks)
    dims = _validate(q, k, v)
    for name, t in (("o", o), ("do", do)):
        if not isinstance(t, torch.Tensor) or t.shape != q.shape or t.dtype != q.dtype:
            raise ValueError(f"{name} must have q's shape {tuple(q.shape)} and dtype {q.dtype}")
        _check_rows(t, name)
    if not isinstance(lse, torch.Tensor) or lse.shape != q.shape[:3] or lse.dtype != torch.float32 or \
            not lse.is_contiguous():
        raise ValueError(f"lse must be the float32 {tuple(q.shape[:3])} tensor that window_attn returned")
    _check_devices(q, o, lse, do)
    P = _params(q, k, v, *dims, n_seq, w, s, scale)
    B, T, S, Hq, Hk, D = dims
    P.o_stride[:], P.do_stride[:] = o.stride()[:3], do.stride()[:3]
    P.dq_stride[:] = (T * Hq * D, Hq * D, D)
    P.dk_stride[:] = P.dv_stride[:] = (S * Hk * D, Hk * D, D)
    P.cu_seqlens = 1 if n_seq is not None else None     # only whether it is set counts here
    ws = _lib.load_library().gdn_attn_bwd_workspace_size(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"window_attn_bwd does not support q {tuple(q.shape)}, k {tuple(k.shape)}")
    P.cu_seqlens = None
    return bytes(P), int(ws)


def _run_bwd(q, k, v, o, lse, do, window, sinks, scale, cu, n_seq):
    # autograd may hand over any layout, e.g. the expansion of a scalar
    if isinstance(do, torch.Tensor) and do.dim() == 4 and do.numel() > 0 and \
            (do.stride(-1) != 1 or do.data_ptr() % 16 or any(s % 8 for s in do.stride()[:3])):
        do = do.clone(memory_format=torch.contiguous_format)
    try:
        key = (_sig(q), _sig(k), _sig(v), _sig(o), _sig(lse), _sig(do), window, sinks, scale, n_seq)
        plan = _BWD_PLANS.get(key)
    except (AttributeError, TypeError):
        key, plan = None, None
    if plan is None:
        plan = _bwd_plan(q, k, v, o, lse, do, window, sinks, scale, n_seq)
        if key is not None:
            if len(_BWD_PLANS) >= _PLANS_MAX:
                _BWD_PLANS.clear()
            _BWD_PLANS[key] = plan
    elif not _aligned(q, k, v, o, do):
        _bwd_plan(q, k, v, o, lse, do, window, sinks, scale, n_seq)
    params, ws_bytes = plan
    dev = q.device
    dq, dk, dv = _like(q), _like(k), _like(v)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    P = _lib.GdnAttnParams.from_buffer_copy(params)
    P.q, P.k, P.v, P.o, P.lse, P.d_o = (t.data_ptr() for t in (q, k, v, o, lse, do))
    P.dq, P.dk, P.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    P.cu_seqlens = cu.data_ptr() if cu is not None else None
    P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_attn_bwd_launch, P, dev)
    if status != 0:
        raise _failed("gdn_attn_bwd_launch", status)
    return dq, dk, dv


def window_attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                    do: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                    scale: Optional[float] = None, *, cu_seqlens: Optional[torch.Tensor] = None):
    """Gradients ``(dq, dk, dv)`` of ``window_attn`` given ``do`` (of ``o``), the
    ``o`` and ``lse`` that it returned and the same other arguments.  A key
    head's gradient is the sum over the query heads that share it, in a fixed
    order: repeated calls give the same bits."""
    cu, n_seq = _seqs(q, cu_seqlens)
    return _run_bwd(q, k, v, o, lse, do, window, sinks, _number(scale), cu, n_seq)


class _AttnFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, cu, n_seq):
        o, lse = _run(q, k, v, window, sinks, scale, cu, n_seq, True)
        ctx.save_for_backward(q, k, v, o, lse, cu)
        ctx.mark_non_differentiable(lse)
        ctx.window, ctx.sinks, ctx.scale = window, sinks, scale
        return o, lse

    @staticmethod
    @_first_order
    def backward(ctx, do, _):
        q, k, v, o, lse, cu = ctx.saved_tensors
        n_seq = None
        if cu is not None:
            cu, n_seq = _offsets(cu, q.device)      # saved-tensor hooks may hand back another
        dq, dk, dv = _run_bwd(q, k, v, o, lse, do, ctx.window, ctx.sinks, ctx.scale, cu, n_seq)
        return dq, dk, dv, None, None, None, None, None


def _decode_plan(q, k_cache, v_cache, lens, window, sinks, scale):
    w, s = _check_window(window, sinks)
    B, T, S, Hq, Hk, D = _validate(q, k_cache, v_cache, ("q", "k_cache", "v_cache"))
    if not 1 <= T <= MAX_DECODE_T:
        raise ValueError(f"q must hold 1 to {MAX_DECODE_T} new tokens of each sequence, got {T}")
    if S < 1:
        raise ValueError("the cache has no rows")
    if not isinstance(lens, torch.Tensor) or tuple(lens.shape) != (B,) or lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cache_seqlens must be an int32 or int64 tensor of [B] = [{B}]")
    _check_devices(q, lens)
    P = _lib.GdnAttnDecodeParams()
    P.B, P.T, P.S, P.Hq, P.Hk, P.D = B, T, S, Hq, Hk, D
    P.window, P.sinks = w, s
    P.scale = D ** -0.5 if scale is None else scale
    P.dtype = _DTYPE_CODE[q.dtype]
    P.q_stride[:], P.k_stride[:], P.v_stride[:] = q.stride()[:3], k_cache.stride()[:3], v_cache.stride()[:3]
    P.o_stride[:] = (T * Hq * D, Hq * D, D)
    ws = _lib.load_library().gdn_attn_decode_workspace_size(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"window_attn_decode does not support q {tuple(q.shape)}, cache {tuple(k_cache.shape)}")
    return bytes(P), int(ws)


def window_attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       cache_seqlens: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                       scale: Optional[float] = None) -> torch.Tensor:
    """``window_attn`` for the newest tokens of B running sequences.

    Args:
      q: ``[B, T, Hq, D]``, 1 to 16 new tokens of each sequence.
      k_cache, v_cache: ``[B, S, Hk, D]``; the first ``cache_seqlens[b]`` rows
        are sequence b's keys, the new tokens' own rows (written by the
        caller) the last T of them.  Rows from there on are never read.
      cache_seqlens: ``[B]`` int32 (or int64) on the device, not read on the
        host; the kernel clamps it to ``[0, S]``.  A token that stands before
        the first key gives zero.

    Returns ``o [B, T, Hq, D]``.  Not differentiable.
    """
    if _needs_grad(q, k_cache, v_cache):
        raise NotImplementedError("window_attn_decode has no gradient: use window_attn in training")
    scale = _number(scale)
    try:
        key = (_sig(q), _sig(k_cache), _sig(v_cache), _sig(cache_seqlens), window, sinks, scale)
        plan = _DECODE_PLANS.get(key)
    except (AttributeError, TypeError):
        key, plan = None, None
    if plan is None:
        plan = _decode_plan(q, k_cache, v_cache, cache_seqlens, window, sinks, scale)
        if key is not None:
            if len(_DECODE_PLANS) >= _PLANS_MAX:
                _DECODE_PLANS.clear()
            _DECODE_PLANS[key] = plan
    elif not _aligned(q, k_cache, v_cache):
        _validate(q, k_cache, v_cache, ("q", "k_cache", "v_cache"))
    params, ws_bytes = plan
    lens = cache_seqlens
    if lens.dtype != torch.int32 or not lens.is_contiguous():
        lens = lens.clamp(0, k_cache.shape[1]).to(torch.int32).contiguous()
    o = _like(q)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes > 0 else None
    P = _lib.GdnAttnDecodeParams.from_buffer_copy(params)
    P.q, P.k, P.v, P.o = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr()
    P.cache_seqlens = lens.data_ptr()
    if ws is not None:
        P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_attn_decode_launch, P, q.device)
    if status != 0:
        raise _failed("gdn_attn_decode_launch", status)
    return o
