"""MI355X-native fused chunked Gated DeltaNet forward.

The hot path of ``v100-attention-lab`` (``gdn_chunk_fwd``,
gdn_triton.py:113-140) as a hand-written gfx950 HIP kernel behind a C ABI
(``include/gdn_mi355x.h``), called from PyTorch-ROCm through ctypes, and the
operators that a hybrid model runs beside it: ``gated_scan`` (an elementwise
gated recurrence), ``window_attn`` (softmax attention with a sliding window and
sinks) and ``add_rms_norm``, with their backward and single-token forms; the
head's loss ``linear_xent``; and for serving ``fp8_linear`` and an 8-bit key and
value cache (``cache_write_fp8``, ``window_attn_decode_fp8``).

The directory name is not a Python identifier; import it with
``importlib.import_module("v100-attention-lab_amd")`` -- it also registers
itself as ``v100_attention_lab_amd``.
"""

import sys as _sys

from ._lib import load_library, status_string, LIB_PATH  # noqa: F401
from .ops import (gdn_fwd, gdn_chunk_fwd, auto_block_v, gdn_prep, l2norm,  # noqa: F401
                  chunk_gated_delta_rule, gdn_bwd)
from .scan import gated_scan, gated_scan_bwd  # noqa: F401
from .attn import window_attn, window_attn_bwd, window_attn_decode  # noqa: F401
from .norm import add_rms_norm, add_rms_norm_bwd, add_rms_norm_fp8  # noqa: F401
from .cache import cache_read_fp8, cache_write_fp8, window_attn_decode_fp8  # noqa: F401
from .linear import fp8_linear, quantize_fp8, quantize_fp8_weight  # noqa: F401
from .loss import linear_xent, linear_xent_bwd  # noqa: F401

_sys.modules.setdefault("v100_attention_lab_amd", _sys.modules[__name__])

__all__ = ["gdn_fwd", "gdn_chunk_fwd", "chunk_gated_delta_rule", "gdn_prep", "l2norm",
           "gdn_bwd", "auto_block_v", "gated_scan", "gated_scan_bwd", "add_rms_norm", "add_rms_norm_bwd",
           "add_rms_norm_fp8", "window_attn", "window_attn_bwd", "window_attn_decode",
           "linear_xent", "linear_xent_bwd", "fp8_linear", "quantize_fp8", "quantize_fp8_weight",
           "cache_write_fp8", "cache_read_fp8", "window_attn_decode_fp8", "load_library", "status_string"]
