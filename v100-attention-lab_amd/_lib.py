"""ctypes binding of the C ABI declared in ``include/gdn_mi355x.h``."""

from __future__ import annotations

import ctypes
import os
import threading

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG_DIR, "lib", "libgdn_mi355x.so")

ABI_VERSION = 5

# enum GdnDtype
DTYPE_F32 = 0
DTYPE_F16 = 1
DTYPE_BF16 = 2

# enum GdnStatus (argument errors; other non-zero values are hipError_t)
GDN_OK = 0
GDN_ERR_NULL_POINTER = 1001
GDN_ERR_BAD_SHAPE = 1002
GDN_ERR_UNSUPPORTED = 1003
GDN_ERR_MISALIGNED = 1004
GDN_ERR_BAD_DTYPE = 1005
GDN_ERR_WORKSPACE = 1006
GDN_ERR_SCRATCH_LIMIT = 1007

# enum GdnFp8Mode
FP8_GROUPS = 0
FP8_ROWS = 1
FP8_BLOCKS = 2

# enum GdnFlags
FLAG_PHASED_KERNEL = 1
FLAG_FUSED_KERNEL = 2

# Every symbol the header declares; tests check the library exports them.
EXPORTED_SYMBOLS = (
    "gdn_fwd_launch",
    "gdn_fwd_workspace_size",
    "gdn_fwd_auto_block_v",
    "gdn_fwd_status_string",
    "gdn_fwd_abi_version",
    "gdn_prep_launch",
    "gdn_bwd_workspace_size",
    "gdn_bwd_workspace_size_params",
    "gdn_bwd_segment_workspace_size",
    "gdn_bwd_launch",
    "gdn_fwd_launch_noalloc",
    "gdn_fwd_scratch_bytes",
    "gdn_scan_chunk",
    "gdn_scan_slots",
    "gdn_scan_workspace_size",
    "gdn_scan_bwd_workspace_size",
    "gdn_scan_launch",
    "gdn_scan_bwd_launch",
    "gdn_norm_launch",
    "gdn_norm_bwd_workspace_size",
    "gdn_norm_bwd_launch",
    "gdn_attn_workspace_size",
    "gdn_attn_launch",
    "gdn_attn_bwd_workspace_size",
    "gdn_attn_bwd_launch",
    "gdn_attn_decode_workspace_size",
    "gdn_attn_decode_launch",
    "gdn_xent_workspace_size",
    "gdn_xent_launch",
    "gdn_xent_bwd_workspace_size",
    "gdn_xent_bwd_launch",
    "gdn_fp8_quant_launch",
    "gdn_fp8_linear_launch",
    "gdn_cache8_write_launch",
    "gdn_cache8_read_launch",
    "gdn_cache8_decode_workspace_size",
    "gdn_cache8_decode_launch",
)

_I64x2 = ctypes.c_int64 * 2
_I64x3 = ctypes.c_int64 * 3
_I64x4 = ctypes.c_int64 * 4


class GdnFwdParams(ctypes.Structure):
    """Mirror of ``struct GdnFwdParams`` (field order and types match)."""

    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("g", ctypes.c_void_p),
        ("beta", ctypes.c_void_p),
        ("h0", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("final_state", ctypes.c_void_p),
        ("q_stride", _I64x3),
        ("k_stride", _I64x3),
        ("v_stride", _I64x3),
        ("g_stride", _I64x3),
        ("beta_stride", _I64x3),
        ("o_stride", _I64x3),
        ("h0_stride", _I64x4),
        ("fs_stride", _I64x4),
        ("B", ctypes.c_int32),
        ("T", ctypes.c_int32),
        ("H", ctypes.c_int32),
        ("K", ctypes.c_int32),
        ("V", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("chunk_size", ctypes.c_int32),
        ("block_v", ctypes.c_int32),
        ("qkv_dtype", ctypes.c_int32),
        ("g_dtype", ctypes.c_int32),
        ("beta_dtype", ctypes.c_int32),
        ("o_dtype", ctypes.c_int32),
        ("flags", ctypes.c_int32),
        ("cu_seqlens", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
    ]


class GdnPrepParams(ctypes.Structure):
    """Mirror of ``GdnPrepParams`` in include/gdn_mi355x.h."""

    _fields_ = [
        ("q_in", ctypes.c_void_p),
        ("q_out", ctypes.c_void_p),
        ("k_in", ctypes.c_void_p),
        ("k_out", ctypes.c_void_p),
        ("beta_in", ctypes.c_void_p),
        ("beta_out", ctypes.c_void_p),
        ("g_in", ctypes.c_void_p),
        ("g_out", ctypes.c_void_p),
        ("q_in_stride", _I64x3),
        ("q_out_stride", _I64x3),
        ("k_in_stride", _I64x3),
        ("k_out_stride", _I64x3),
        ("beta_in_stride", _I64x3),
        ("beta_out_stride", _I64x3),
        ("g_in_stride", _I64x3),
        ("g_out_stride", _I64x3),
        ("B", ctypes.c_int32),
        ("T", ctypes.c_int32),
        ("H", ctypes.c_int32),
        ("K", ctypes.c_int32),
        ("qk_dtype", ctypes.c_int32),
        ("beta_in_dtype", ctypes.c_int32),
        ("beta_out_dtype", ctypes.c_int32),
        ("g_in_dtype", ctypes.c_int32),
        ("g_out_dtype", ctypes.c_int32),
        ("eps", ctypes.c_float),
    ]


class GdnBwdParams(ctypes.Structure):
    """Mirror of ``GdnBwdParams`` in include/gdn_mi355x.h."""

    _fields_ = [(n, ctypes.c_void_p) for n in (
        "q", "k", "v", "g", "beta", "h0", "d_o", "d_final_state",
        "dq", "dk", "dv", "dg", "dbeta", "dh0", "workspace")] + \
        [(n, _I64x3) for n in (
            "q_stride", "k_stride", "v_stride", "g_stride", "beta_stride", "do_stride",
            "dq_stride", "dk_stride", "dv_stride", "dg_stride", "dbeta_stride")] + \
        [(n, _I64x4) for n in ("h0_stride", "dfs_stride", "dh0_stride")] + \
        [(n, ctypes.c_int32) for n in ("B", "T", "H", "K", "V")] + \
        [("scale", ctypes.c_float)] + \
        [(n, ctypes.c_int32) for n in ("qkv_dtype", "g_dtype", "beta_dtype", "do_dtype")] + \
        [("cu_seqlens", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)]


def _fields(*groups):
    """(name, type) pairs of groups of names with one type each."""
    return [(n, t) for names, t in groups for n in names.split()]


class GdnScanParams(ctypes.Structure):
    """Mirror of ``GdnScanParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("x g h0 y final_state states dy dfinal dx dg dh0 cu_seqlens workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
        ("x_stride g_stride y_stride dy_stride dx_stride dg_stride", _I64x2),
        ("h0_stride dfinal_stride", ctypes.c_int64),
        ("B T D N x_dtype g_dtype", ctypes.c_int32))


class GdnNormParams(ctypes.Structure):
    """Mirror of ``GdnNormParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("x res w y r_out scale r dy dr_in dr dx dw workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
        ("x_stride res_stride y_stride r_out_stride r_stride dy_stride dr_in_stride dr_stride dx_stride", _I64x2),
        ("n_outer n_inner D", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("group x_dtype r_dtype w_dtype", ctypes.c_int32))


class GdnAttnParams(ctypes.Structure):
    """Mirror of ``GdnAttnParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("q k v o lse d_o dq dk dv cu_seqlens workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
        ("q_stride k_stride v_stride o_stride do_stride dq_stride dk_stride dv_stride", _I64x3),
        ("B Tq Tk N Hq Hk D window sinks", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("dtype", ctypes.c_int32))


class GdnAttnDecodeParams(ctypes.Structure):
    """Mirror of ``GdnAttnDecodeParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("q k v o cache_seqlens workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
        ("q_stride k_stride v_stride o_stride", _I64x3),
        ("B T S Hq Hk D window sinks", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("dtype", ctypes.c_int32))


class GdnXentParams(ctypes.Structure):
    """Mirror of ``GdnXentParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("x w target loss lse dloss dx dw workspace", ctypes.c_void_p),
        ("workspace_bytes x_stride w_stride dloss_stride", ctypes.c_int64),
        ("N D V dtype", ctypes.c_int32))


class GdnFp8QuantParams(ctypes.Structure):
    """Mirror of ``GdnFp8QuantParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("x q scale", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64),
        ("rows D x_dtype mode", ctypes.c_int32))


class GdnFp8LinearParams(ctypes.Structure):
    """Mirror of ``GdnFp8LinearParams`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("x x_scale w w_scale y", ctypes.c_void_p),
        ("x_stride w_stride", ctypes.c_int64),
        ("M N K group y_dtype", ctypes.c_int32))


class GdnCache8Params(ctypes.Structure):
    """Mirror of ``GdnCache8Params`` in include/gdn_mi355x.h."""

    _fields_ = _fields(
        ("k v q o k_cache v_cache k_scale v_scale cache_seqlens workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
        ("k_stride v_stride q_stride o_stride kc_stride vc_stride ks_stride vs_stride", _I64x3),
        ("B T S Hq Hk D window sinks", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("dtype", ctypes.c_int32))


_lock = threading.Lock()
_lib = None


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the built HIP library (once).  Raises ImportError if it is missing.

    There is no fallback: without the library the GDN forward is unavailable.
    """
    global _lib
    if _lib is not None:        # (set once, whole)
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(path):
            raise ImportError(
                f"GDN HIP library not found at {path}; build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` or "
                "`python v100-attention-lab_amd/build.py`")
        lib = ctypes.CDLL(path)
        lib.gdn_fwd_launch.argtypes = [ctypes.POINTER(GdnFwdParams), ctypes.c_void_p]
        lib.gdn_fwd_launch.restype = ctypes.c_int
        lib.gdn_fwd_launch_noalloc.argtypes = [ctypes.POINTER(GdnFwdParams), ctypes.c_void_p]
        lib.gdn_fwd_launch_noalloc.restype = ctypes.c_int
        lib.gdn_fwd_scratch_bytes.argtypes = []
        lib.gdn_fwd_scratch_bytes.restype = ctypes.c_int64
        lib.gdn_fwd_workspace_size.argtypes = [ctypes.POINTER(GdnFwdParams)]
        lib.gdn_fwd_workspace_size.restype = ctypes.c_int64
        lib.gdn_fwd_auto_block_v.argtypes = [ctypes.c_int] * 6
        lib.gdn_fwd_auto_block_v.restype = ctypes.c_int
        lib.gdn_fwd_status_string.argtypes = [ctypes.c_int]
        lib.gdn_fwd_status_string.restype = ctypes.c_char_p
        lib.gdn_prep_launch.argtypes = [ctypes.POINTER(GdnPrepParams), ctypes.c_void_p]
        lib.gdn_prep_launch.restype = ctypes.c_int
        lib.gdn_bwd_launch.argtypes = [ctypes.POINTER(GdnBwdParams), ctypes.c_void_p]
        lib.gdn_bwd_launch.restype = ctypes.c_int
        lib.gdn_bwd_workspace_size.argtypes = [ctypes.c_int] * 6
        lib.gdn_bwd_workspace_size.restype = ctypes.c_int64
        lib.gdn_bwd_workspace_size_params.argtypes = [ctypes.POINTER(GdnBwdParams)]
        lib.gdn_bwd_workspace_size_params.restype = ctypes.c_int64
        lib.gdn_bwd_segment_workspace_size.argtypes = [ctypes.POINTER(GdnBwdParams), ctypes.c_int]
        lib.gdn_bwd_segment_workspace_size.restype = ctypes.c_int64
        for name, struct in (("scan", GdnScanParams), ("scan_bwd", GdnScanParams), ("norm", GdnNormParams),
                             ("norm_bwd", GdnNormParams), ("attn", GdnAttnParams), ("attn_bwd", GdnAttnParams),
                             ("attn_decode", GdnAttnDecodeParams), ("xent", GdnXentParams),
                             ("xent_bwd", GdnXentParams), ("fp8_quant", GdnFp8QuantParams),
                             ("fp8_linear", GdnFp8LinearParams), ("cache8_write", GdnCache8Params),
                             ("cache8_read", GdnCache8Params), ("cache8_decode", GdnCache8Params)):
            if f"gdn_{name}_workspace_size" in EXPORTED_SYMBOLS:
                size = getattr(lib, f"gdn_{name}_workspace_size")
                size.argtypes, size.restype = [ctypes.POINTER(struct)], ctypes.c_int64
            launch = getattr(lib, f"gdn_{name}_launch")
            launch.argtypes, launch.restype = [ctypes.POINTER(struct), ctypes.c_void_p], ctypes.c_int
        lib.gdn_scan_chunk.argtypes = []
        lib.gdn_scan_chunk.restype = ctypes.c_int
        lib.gdn_scan_slots.argtypes = [ctypes.c_int] * 4
        lib.gdn_scan_slots.restype = ctypes.c_int64
        lib.gdn_fwd_abi_version.argtypes = []
        lib.gdn_fwd_abi_version.restype = ctypes.c_int
        ver = lib.gdn_fwd_abi_version()
        if ver != ABI_VERSION:
            raise ImportError(f"{path}: ABI version {ver}, expected {ABI_VERSION}; rebuild")
        _lib = lib
        return lib


def status_string(code: int) -> str:
    return load_library().gdn_fwd_status_string(int(code)).decode()


_OP_STATUS = {
    GDN_ERR_NULL_POINTER: "a required pointer is NULL",
    GDN_ERR_BAD_SHAPE: "invalid sizes",
    GDN_ERR_UNSUPPORTED: "unsupported configuration",
    GDN_ERR_MISALIGNED: "rows must be 16-byte aligned with a contiguous last dimension",
    GDN_ERR_BAD_DTYPE: "unsupported dtypes",
    GDN_ERR_WORKSPACE: "workspace missing, misaligned or too small",
}


def op_status_string(code: int) -> str:
    """Text of a status of the scan, norm and attention calls."""
    return _OP_STATUS.get(code) or status_string(code)
