"""A key and value cache in e4m3 with a scale for each row and head: writing it,
reading it back, and windowed attention of the newest tokens over it
(``csrc/gdn_cache8.hip``).  No counterpart in the reference."""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .attn import MAX_DECODE_T, SUPPORTED_D, _check_window, _number
from .ops import _DTYPE_CODE, _PLANS_MAX, _check_devices, _check_sizes, _code, _launch, _needs_grad
from .scan import _failed, _like, _sig

FP8 = torch.float8_e4m3fn

_PLANS = {}


def _check_rows(t, name):
    """Rows are read 16 bytes at a time; strides of single indexes do not count."""
    if t.numel() == 0:
        return
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous (stride {t.stride(-1)}); "
                         "call .contiguous()")
    if t.data_ptr() % 16 != 0 or any(s * t.element_size() % 16 for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1):
        raise ValueError(f"{name}: rows must be 16-byte aligned (data_ptr and strides {t.stride()[:3]}); "
                         "call .contiguous()")


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype != FP8:
            raise ValueError(f"{name} must be a float8_e4m3fn [B, S, Hk, D] tensor")
    B, S, Hk, D = k_cache.shape
    if v_cache.shape != k_cache.shape:
        raise ValueError(f"v_cache {tuple(v_cache.shape)} must have k_cache's shape {tuple(k_cache.shape)}")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if not isinstance(t, torch.Tensor) or tuple(t.shape) != (B, S, Hk) or t.dtype != torch.float32:
            raise ValueError(f"{name} must be float32 [B, S, Hk] = {(B, S, Hk)}")
    if D not in SUPPORTED_D:
        raise ValueError(f"D={D} not supported (D in {SUPPORTED_D})")
    if B <= 0 or S <= 0 or Hk <= 0:
        raise ValueError(f"the cache has no rows: {tuple(k_cache.shape)}")
    if k_cache.device.type != "cuda":
        raise ValueError(f"the 8-bit cache lives on a ROCm GPU (got {k_cache.device}); there is no CPU path")
    _check_devices(k_cache, v_cache, k_scale, v_scale)
    _check_sizes(*k_cache.shape)
    _check_rows(k_cache, "k_cache")
    _check_rows(v_cache, "v_cache")
    return B, S, Hk, D


def _check_lens(lens, cache):
    B = cache.shape[0]
    if not isinstance(lens, torch.Tensor) or tuple(lens.shape) != (B,) or lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cache_seqlens must be an int32 or int64 tensor of [B] = [{B}]")
    _check_devices(cache, lens)


def _lens32(lens, S):
    if lens.dtype != torch.int32 or not lens.is_contiguous():
        lens = lens.clamp(0, S).to(torch.int32).contiguous()
    return lens


def _params(k_cache, v_cache, k_scale, v_scale, B, S, Hk, D):
    P = _lib.GdnCache8Params()
    P.B, P.S, P.Hk, P.D = B, S, Hk, D
    P.kc_stride[:], P.vc_stride[:] = k_cache.stride()[:3], v_cache.stride()[:3]
    P.ks_stride[:], P.vs_stride[:] = k_scale.stride(), v_scale.stride()
    return P


def _call(what, rows, others, options, make):
    """The plan of a signature seen before, or make()'s.  (The alignment of `rows` is
    of this call's pointers: part of the signature.)"""
    try:
        key, bits = [what, options], 0
        for t in rows:
            bits |= t.data_ptr()
            key.append(_sig(t))
        for t in others:
            key.append(_sig(t))
        key = (*key, bits & 15)
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):     # not tensors: the checks say which
        key, plan = None, None
    if plan is None:
        plan = make()
        if key is not None:
            if len(_PLANS) >= _PLANS_MAX:
                _PLANS.clear()
            _PLANS[key] = plan
    return plan


def _bind(params, k_cache, v_cache, k_scale, v_scale):
    P = _lib.GdnCache8Params.from_buffer_copy(params)
    P.k_cache, P.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    P.k_scale, P.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    return P


def _write_plan(k, v, k_cache, v_cache, k_scale, v_scale, lens):
    B, S, Hk, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale)):
        if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise ValueError(f"{name} is written to and must not be expanded (strides {t.stride()})")
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or (t.shape[0], *t.shape[2:]) != (B, Hk, D):
            raise ValueError(f"{name} must be [B, T, Hk, D] with the cache's B={B}, Hk={Hk}, D={D}")
        _code(t, name)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"k and v must share shape and dtype (got {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype})")
    _check_lens(lens, k_cache)
    _check_devices(k_cache, k, v)
    _check_rows(k, "k")
    _check_rows(v, "v")
    _check_sizes(k.shape[1])
    P = _params(k_cache, v_cache, k_scale, v_scale, B, S, Hk, D)
    P.T, P.dtype = k.shape[1], _DTYPE_CODE[k.dtype]
    P.k_stride[:], P.v_stride[:] = k.stride()[:3], v.stride()[:3]
    return bytes(P)


def cache_write_fp8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, cache_seqlens: torch.Tensor) -> None:
    """Writes the newest T rows of B sequences into their caches, in 8 bits.

    Args:
      k, v: ``[B, T, Hk, D]`` float16, bfloat16 or float32, D in {64, 128},
        16-byte aligned rows, any other strides; any T (a token, a prompt).
      k_cache, v_cache: ``[B, S, Hk, D]`` float8_e4m3fn; k_scale, v_scale:
        ``[B, S, Hk]`` float32.  Row i of the new ones becomes row
        ``cache_seqlens[b] - T + i`` of sequence b: ``max|x| / 448`` over its D
        columns goes into the scale and ``x / scale``, rounded, into the cache.
        Rows that would lie before the first (the padding in front of a shorter
        prompt) are dropped, all other rows are left as they are.
      cache_seqlens: ``[B]`` int32 (or int64) on the device, the new tokens
        among them, as ``window_attn_decode_fp8`` takes it; not read on the
        host, clamped to ``[0, S]``.

    Not differentiable.
    """
    if _needs_grad(k, v, k_scale, v_scale):
        raise NotImplementedError("cache_write_fp8 has no gradient")
    params = _call("write", (k, v, k_cache, v_cache), (k_scale, v_scale, cache_seqlens), None,
                   lambda: _write_plan(k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens))
    if k.shape[1] == 0:
        return
    lens = _lens32(cache_seqlens, k_cache.shape[1])
    P = _bind(params, k_cache, v_cache, k_scale, v_scale)
    P.k, P.v, P.cache_seqlens = k.data_ptr(), v.data_ptr(), lens.data_ptr()
    status = _launch(_lib.load_library().gdn_cache8_write_launch, P, k_cache.device)
    if status != 0:
        raise _failed("gdn_cache8_write_launch", status)


def _read_plan(k_cache, v_cache, k_scale, v_scale, dtype):
    B, S, Hk, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"dtype {dtype} not supported (float32, float16, bfloat16)")
    P = _params(k_cache, v_cache, k_scale, v_scale, B, S, Hk, D)
    P.dtype = _DTYPE_CODE[dtype]
    P.k_stride[:] = P.v_stride[:] = (S * Hk * D, Hk * D, D)
    return bytes(P)


def cache_read_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, *,
                   dtype: torch.dtype = torch.bfloat16):
    """``(k, v)`` of an 8-bit cache (see ``cache_write_fp8``) in ``dtype``,
    ``[B, S, Hk, D]`` each: every byte times its row's scale, rounded once.
    Part of a cache is read from slices of all four tensors, e.g. ``[:, :n]``
    for the keys that a prefill continues."""
    if _needs_grad(k_scale, v_scale):
        raise NotImplementedError("cache_read_fp8 has no gradient")
    params = _call("read", (k_cache, v_cache), (k_scale, v_scale), dtype,
                   lambda: _read_plan(k_cache, v_cache, k_scale, v_scale, dtype))
    k = torch.empty(k_cache.shape, dtype=dtype, device=k_cache.device)
    v = torch.empty_like(k)
    P = _bind(params, k_cache, v_cache, k_scale, v_scale)
    P.k, P.v = k.data_ptr(), v.data_ptr()
    status = _launch(_lib.load_library().gdn_cache8_read_launch, P, k_cache.device)
    if status != 0:
        raise _failed("gdn_cache8_read_launch", status)
    return k, v


def _decode_plan(q, k_cache, v_cache, k_scale, v_scale, lens, window, sinks, scale):
    w, s = _check_window(window, sinks)
    B, S, Hk, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[0] != B or q.shape[3] != D:
        raise ValueError(f"q must be [B, T, Hq, D] with the cache's B={B} and D={D}")
    T, Hq = q.shape[1:3]
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q must be float16 or bfloat16, got {q.dtype}")
    if Hq <= 0 or Hq % Hk != 0:
        raise ValueError(f"Hq={Hq} must be a positive multiple of Hk={Hk}")
    if not 1 <= T <= MAX_DECODE_T:
        raise ValueError(f"q must hold 1 to {MAX_DECODE_T} new tokens of each sequence, got {T}")
    _check_lens(lens, k_cache)
    _check_devices(k_cache, q)
    _check_sizes(Hq)
    _check_rows(q, "q")
    P = _params(k_cache, v_cache, k_scale, v_scale, B, S, Hk, D)
    P.T, P.Hq, P.window, P.sinks = T, Hq, w, s
    P.scale = D ** -0.5 if scale is None else scale
    P.dtype = _DTYPE_CODE[q.dtype]
    P.q_stride[:] = q.stride()[:3]
    P.o_stride[:] = (T * Hq * D, Hq * D, D)
    ws = _lib.load_library().gdn_cache8_decode_workspace_size(ctypes.byref(P))
    if ws < 0:
        raise ValueError(f"window_attn_decode_fp8 does not support q {tuple(q.shape)}, cache {tuple(k_cache.shape)}")
    return bytes(P), int(ws)


def window_attn_decode_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                           v_scale: torch.Tensor, cache_seqlens: torch.Tensor, window: Optional[int] = None,
                           sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """``window_attn_decode`` over an 8-bit cache: keys ``k_cache * k_scale`` and
    values ``v_cache * v_scale``.

    Args:
      q: ``[B, T, Hq, D]`` float16 or bfloat16, 1 to 16 new tokens of each
        sequence, whose own rows ``cache_write_fp8`` has put into the cache.
      k_cache, v_cache, k_scale, v_scale, cache_seqlens: as
        ``cache_write_fp8`` takes them; rows from ``cache_seqlens[b]`` on are
        never read.
      window, sinks, scale: as in ``window_attn``.

    Returns ``o [B, T, Hq, D]`` in q's dtype.  Not differentiable.
    """
    if _needs_grad(q, k_scale, v_scale):
        raise NotImplementedError("window_attn_decode_fp8 has no gradient: use window_attn in training")
    scale = _number(scale)
    params, ws_bytes = _call(
        "decode", (q, k_cache, v_cache), (k_scale, v_scale, cache_seqlens), (window, sinks, scale),
        lambda: _decode_plan(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, window, sinks, scale))
    lens = _lens32(cache_seqlens, k_cache.shape[1])
    o = _like(q)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes > 0 else None
    P = _bind(params, k_cache, v_cache, k_scale, v_scale)
    P.q, P.o, P.cache_seqlens = q.data_ptr(), o.data_ptr(), lens.data_ptr()
    if ws is not None:
        P.workspace, P.workspace_bytes = ws.data_ptr(), ws_bytes
    status = _launch(_lib.load_library().gdn_cache8_decode_launch, P, q.device)
    if status != 0:
        raise _failed("gdn_cache8_decode_launch", status)
    return o
