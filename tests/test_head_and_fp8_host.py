"""CPU tests of linear_xent, the 8-bit product and the 8-bit cache: the ctypes
mirrors against the header, the refusals of the C ABI (nothing is enqueued) and of
the Python surface, and the workspace sizes."""

import ctypes
import os
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(REPO, "include")
FAKE = 0x100000       # never read: every refusal below comes before the launch
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib(pkg):
    if not os.path.exists(pkg.LIB_PATH):
        from importlib import import_module
        import_module("v100-attention-lab_amd.build").build(verbose=False)
    return pkg.load_library()


@pytest.mark.parametrize("struct", ["GdnXentParams", "GdnFp8QuantParams", "GdnFp8LinearParams", "GdnCache8Params"])
def test_struct_layout_matches_header(tmp_path, pkg, struct):
    S = getattr(pkg._lib, struct)
    fields = [f for f, _ in S._fields_]
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof({struct}, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "gdn_mi355x.h"\nint main(void) {{\n{body}\n'
                   f'  printf("sizeof %zu\\n", sizeof({struct}));\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{INCLUDE}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    layout = dict(zip(out[0::2], map(int, out[1::2])))
    for f in fields:
        assert getattr(S, f).offset == layout[f], f
    assert ctypes.sizeof(S) == layout["sizeof"]


def _fill(P, pointers, values, kw):
    for n in pointers.split():
        setattr(P, n, FAKE)
    for k, v in {**values, **kw}.items():
        if k.endswith("_stride") and isinstance(v, tuple):
            getattr(P, k)[:] = v
        else:
            setattr(P, k, v)
    return P


def _xent(L, **kw):
    return _fill(L.GdnXentParams(), "x w target loss lse dloss dx dw workspace", dict(
        workspace_bytes=1 << 50, x_stride=256, w_stride=256, dloss_stride=1, N=1000, D=256, V=5000,
        dtype=L.DTYPE_BF16), kw)


XENT = [(dict(x=None), 1001), (dict(w=None), 1001), (dict(target=None), 1001), (dict(lse=None), 1001),
        (dict(N=-1), 1002), (dict(V=0), 1002), (dict(D=0), 1002), (dict(N=1 << 26), 1002), (dict(V=1 << 29), 1002),
        (dict(N=(1 << 26) - 1, V=1 << 28), 1002), (dict(D=12), 1003), (dict(x_stride=1 << 23), 1003), (dict(w_stride=-256), 1003),
        (dict(dtype=0), 1005), (dict(x=FAKE + 8), 1004), (dict(w_stride=260), 1004),
        (dict(workspace=None), 1006), (dict(workspace=FAKE + 16), 1006), (dict(workspace_bytes=100), 1006)]


@pytest.mark.parametrize("kw,code", XENT + [(dict(loss=None), 1001)])
def test_xent_refusals(lib, pkg, kw, code):
    assert lib.gdn_xent_launch(ctypes.byref(_xent(pkg._lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", XENT + [(dict(dloss=None), 1001), (dict(dx=None), 1001), (dict(dw=None), 1001),
                                            (dict(N=0), 1002), (dict(dx=FAKE + 4), 1004), (dict(dw=FAKE + 8), 1004)])
def test_xent_bwd_refusals(lib, pkg, kw, code):
    assert lib.gdn_xent_bwd_launch(ctypes.byref(_xent(pkg._lib, **kw)), None) == code


def test_xent_sizes(lib, pkg):
    fwd = lambda **kw: lib.gdn_xent_workspace_size(ctypes.byref(_xent(pkg._lib, **kw)))
    bwd = lambda **kw: lib.gdn_xent_bwd_workspace_size(ctypes.byref(_xent(pkg._lib, **kw)))
    assert fwd(N=0) == 0 and bwd(N=0) > 0 and lib.gdn_xent_launch(ctypes.byref(_xent(pkg._lib, N=0)), None) == 0
    assert fwd(D=12) == bwd(D=12) == lib.gdn_xent_workspace_size(None) == lib.gdn_xent_bwd_workspace_size(None) == -1
    assert lib.gdn_xent_launch(None, None) == 1001 and lib.gdn_xent_bwd_launch(None, None) == 1001
    # 8 bytes a row and at least 128 words; never the logits
    assert fwd(N=8192, V=128000) <= 8192 * (1000 * 8 + 4) + 1024
    # G of a piece, and fp32 sums of dx and of a piece of dw in a part for each share of
    # the card that is empty
    for N, D, V in ((8192, 4096, 128000), (100, 64, 50), (1, 8, 1), (1 << 20, 2048, 32000), (65536, 64, 1000)):
        rows = -(-N // 256) * 256
        size = bwd(N=N, D=D, V=V, x_stride=D, w_stride=D)
        g = max(128 << 20, rows * 256 * 2)
        parts = 4 * (-(-N // 256) * 256) * (-(-D // 256) * 256)
        assert 0 < size <= g + rows * 16 + 1024 + max(parts, 4 * 512 * 128 * 128) + 4 * 512 * 128 * 128


def _quant(L, **kw):
    return _fill(L.GdnFp8QuantParams(), "x q scale", dict(x_stride=256, rows=10, D=256, x_dtype=L.DTYPE_BF16, mode=0), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), 1001), (dict(q=None), 1001), (dict(scale=None), 1001), (dict(rows=-1), 1002), (dict(D=0), 1002),
    (dict(rows=1 << 30, D=1 << 20), 1002), (dict(D=200), 1003), (dict(mode=3), 1003), (dict(mode=-1), 1003),
    (dict(x_dtype=5), 1005), (dict(x=FAKE + 8), 1004), (dict(x_stride=260), 1004), (dict(q=FAKE + 4), 1004)])
def test_quant_refusals(lib, pkg, kw, code):
    assert lib.gdn_fp8_quant_launch(ctypes.byref(_quant(pkg._lib, **kw)), None) == code


def _linear(L, **kw):
    return _fill(L.GdnFp8LinearParams(), "x x_scale w w_scale y", dict(
        x_stride=256, w_stride=256, M=100, N=300, K=256, group=128, y_dtype=L.DTYPE_BF16), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), 1001), (dict(x_scale=None), 1001), (dict(w=None), 1001), (dict(w_scale=None), 1001), (dict(y=None), 1001),
    (dict(M=-1), 1002), (dict(N=0), 1002), (dict(K=0), 1002), (dict(M=1 << 29), 1002), (dict(M=1 << 28, N=1 << 28), 1002), (dict(M=1, N=1 << 28), 1002),
    (dict(K=200), 1003), (dict(group=64), 1003), (dict(x_stride=1 << 24), 1003), (dict(w_stride=-128), 1003),
    (dict(y_dtype=8), 1005), (dict(x=FAKE + 8), 1004), (dict(w_stride=264), 1004), (dict(y=FAKE + 8), 1004)])
def test_linear_refusals(lib, pkg, kw, code):
    assert lib.gdn_fp8_linear_launch(ctypes.byref(_linear(pkg._lib, **kw)), None) == code


def test_no_rows_is_nothing(lib, pkg):
    L = pkg._lib
    assert lib.gdn_fp8_quant_launch(ctypes.byref(_quant(L, rows=0)), None) == 0
    assert lib.gdn_fp8_linear_launch(ctypes.byref(_linear(L, M=0)), None) == 0
    assert lib.gdn_cache8_write_launch(ctypes.byref(_cache(L, T=0)), None) == 0
    for name in ("fp8_quant", "fp8_linear", "cache8_write", "cache8_read", "cache8_decode"):
        assert getattr(lib, f"gdn_{name}_launch")(None, None) == 1001


def _cache(L, **kw):
    return _fill(L.GdnCache8Params(), "k v q o k_cache v_cache k_scale v_scale cache_seqlens workspace", dict(
        workspace_bytes=1 << 50, B=2, T=1, S=4096, Hq=8, Hk=2, D=128, window=4096, sinks=0, scale=0.1, dtype=L.DTYPE_BF16,
        q_stride=(1024, 1024, 128), o_stride=(1024, 1024, 128), k_stride=(256, 256, 128), v_stride=(256, 256, 128),
        kc_stride=(4096 * 256, 256, 128), vc_stride=(4096 * 256, 256, 128), ks_stride=(8192, 2, 1), vs_stride=(8192, 2, 1)), kw)


CACHE = [(dict(k_cache=None), 1001), (dict(v_cache=None), 1001), (dict(k_scale=None), 1001), (dict(v_scale=None), 1001),
         (dict(B=0), 1002), (dict(S=0), 1002), (dict(S=1 << 30), 1002), (dict(Hk=0), 1002), (dict(D=80), 1003),
         (dict(k_cache=FAKE + 8), 1004), (dict(vc_stride=(4096 * 256, 264, 128)), 1004), (dict(dtype=9), 1005)]


@pytest.mark.parametrize("kw,code", CACHE + [(dict(k=None), 1001), (dict(v=None), 1001), (dict(cache_seqlens=None), 1001),
                                             (dict(T=-1), 1002), (dict(k=FAKE + 8), 1004), (dict(v_stride=(256, 256, 130)), 1004),
                                             (dict(B=1 << 20, T=1 << 10), 1002), (dict(T=1 << 30, Hk=4), 1002)])
def test_cache_write_refusals(lib, pkg, kw, code):
    assert lib.gdn_cache8_write_launch(ctypes.byref(_cache(pkg._lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", CACHE + [(dict(k=None), 1001), (dict(v=None), 1001), (dict(k=FAKE + 8), 1004),
                                             (dict(B=1 << 18), 1002)])
def test_cache_read_refusals(lib, pkg, kw, code):
    assert lib.gdn_cache8_read_launch(ctypes.byref(_cache(pkg._lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", CACHE + [
    (dict(q=None), 1001), (dict(o=None), 1001), (dict(cache_seqlens=None), 1001), (dict(T=0), 1002), (dict(T=17), 1002),
    (dict(Hq=7), 1002), (dict(window=0), 1002), (dict(sinks=-1), 1002), (dict(B=1 << 20, Hq=16, Hk=16), 1002),
    (dict(Hq=1 << 28, Hk=1, T=16), 1002), (dict(dtype=0), 1005), (dict(q=FAKE + 8), 1004), (dict(workspace=None), 1006),
    (dict(workspace=FAKE + 16), 1006), (dict(workspace_bytes=64), 1006)])
def test_cache_decode_refusals(lib, pkg, kw, code):
    assert lib.gdn_cache8_decode_launch(ctypes.byref(_cache(pkg._lib, **kw)), None) == code


def test_cache_decode_workspace(lib, pkg):
    size = lambda **kw: lib.gdn_cache8_decode_workspace_size(ctypes.byref(_cache(pkg._lib, **kw)))
    assert size() > 0 and size(B=512) == 0 and size(S=100) == 0
    assert size(D=80) == -1 and lib.gdn_cache8_decode_workspace_size(None) == -1


# ---------------------------------------------------------------------------
# Python surface (everything here is refused before the device matters)
# ---------------------------------------------------------------------------

def _operands():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16)
    t, f = torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    x8, w8 = torch.zeros(4, 256).to(FP8), torch.zeros(300, 256).to(FP8)
    kc = torch.zeros(2, 10, 2, 64).to(FP8)
    ks, lens = torch.zeros(2, 10, 2), torch.ones(2, dtype=torch.int32)
    k = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    return dict(x=x, w=w, t=t, f=f, x8=x8, w8=w8, xs=torch.zeros(4, 2), ws=torch.zeros(3, 2), kc=kc, ks=ks, lens=lens, k=k,
                y=torch.zeros(4, 256))


CALLS = {
    "linear_xent": lambda p, o: p.linear_xent(o["x"], o["w"], o["t"]),
    "linear_xent_bwd": lambda p, o: p.linear_xent_bwd(o["x"], o["w"], o["t"], o["f"], o.get("d", o["f"])),
    "quantize_fp8": lambda p, o: p.quantize_fp8(o["y"], group=o.get("group", 128)),
    "quantize_fp8_weight": lambda p, o: p.quantize_fp8_weight(o["y"]),
    "fp8_linear": lambda p, o: p.fp8_linear(o["x8"], o["xs"], o["w8"], o["ws"], out_dtype=o.get("out", torch.float16)),
    "cache_write_fp8": lambda p, o: p.cache_write_fp8(o["k"], o.get("v", o["k"]), o["kc"], o.get("vc", o["kc"]), o["ks"], o["ks"], o["lens"]),
    "cache_read_fp8": lambda p, o: p.cache_read_fp8(o["kc"], o.get("vc", o["kc"]), o["ks"], o["ks"], dtype=o.get("out", torch.float16)),
    "window_attn_decode_fp8": lambda p, o: p.window_attn_decode_fp8(
        o["k"], o["kc"], o.get("vc", o["kc"]), o["ks"], o["ks"], o["lens"], *o.get("args", ())),
}
Z = torch.zeros


@pytest.mark.parametrize("name", list(CALLS))
def test_cpu_tensors_are_refused(pkg, name):
    with pytest.raises(ValueError, match="GPU"):
        CALLS[name](pkg, _operands())


@pytest.mark.parametrize("name,kw,match", [
    ("linear_xent", dict(x=None), "x must"), ("linear_xent", dict(x=Z(64).bfloat16()), "x must"),
    ("linear_xent", dict(w=Z(100, 32).bfloat16()), "weight must"), ("linear_xent", dict(w=Z(0, 64).bfloat16()), "weight must"),
    ("linear_xent", dict(x=Z(4, 64), w=Z(9, 64)), "float16 or bfloat16"), ("linear_xent", dict(w=Z(100, 64).half()), "share"),
    ("linear_xent", dict(x=Z(4, 12).half(), w=Z(9, 12).half()), "multiple of 8"), ("linear_xent", dict(t=Z(4)), "target"),
    ("linear_xent", dict(t=Z(5).long()), "target"), ("linear_xent", dict(t=[0]), "target"),
    ("linear_xent_bwd", dict(t=Z(5).long()), "target"),
    ("quantize_fp8", dict(y=None), "x must"), ("quantize_fp8", dict(y=Z(4, 200)), "multiple of 128"),
    ("quantize_fp8", dict(y=Z(4, 256).long()), "dtype"), ("quantize_fp8", dict(group=64), "group"),
    ("quantize_fp8_weight", dict(y=Z(2, 4, 256)), r"\[N, K\]"), ("quantize_fp8_weight", dict(y=Z(4, 100)), "multiple of 128"),
    ("fp8_linear", dict(x8=Z(4, 256)), "x must"), ("fp8_linear", dict(w8=Z(300, 256)), "weight must"),
    ("fp8_linear", dict(w8=Z(300, 128).to(FP8)), "weight must"), ("fp8_linear", dict(xs=Z(4, 3)), "x_scale"),
    ("fp8_linear", dict(xs=Z(4, 2).half()), "x_scale"), ("fp8_linear", dict(ws=Z(2, 2)), "weight_scale"),
    ("fp8_linear", dict(out=torch.int8), "out_dtype"), ("fp8_linear", dict(x8=Z(4, 100).to(FP8), w8=Z(9, 100).to(FP8)), "multiple"),
    ("cache_write_fp8", dict(kc=Z(2, 10, 2, 64)), "k_cache"), ("cache_write_fp8", dict(vc=Z(2, 9, 2, 64).to(FP8)), "v_cache"),
    ("cache_write_fp8", dict(ks=Z(2, 10)), "k_scale"), ("cache_read_fp8", dict(ks=Z(2, 10, 2).half()), "k_scale"),
    ("cache_read_fp8", dict(kc=Z(2, 10, 2, 80).to(FP8)), "D=80"), ("cache_read_fp8", dict(kc=Z(2, 0, 2, 64).to(FP8), ks=Z(2, 0, 2)), "no rows"),
])
def test_python_refusals(pkg, name, kw, match):
    with pytest.raises(ValueError, match=match):
        CALLS[name](pkg, {**_operands(), **kw})


@pytest.fixture
def as_if_on_gpu(pkg, monkeypatch):
    """The checks behind the device's, on CPU tensors."""
    cache = __import__("importlib").import_module("v100-attention-lab_amd.cache")

    def check(k_cache, *rest):
        B, S, Hk, D = k_cache.shape
        return B, S, Hk, D
    monkeypatch.setattr(cache, "_check_cache", check)
    monkeypatch.setattr(cache, "_check_devices", lambda *ts: None)


@pytest.mark.parametrize("name,kw,match", [
    ("cache_write_fp8", dict(k=Z(2, 1, 3, 64).half()), "k must"), ("cache_write_fp8", dict(v=Z(2, 2, 2, 64).bfloat16()), "share"),
    ("cache_write_fp8", dict(k=Z(2, 1, 2, 64).long()), "dtype"), ("cache_write_fp8", dict(lens=Z(3).int()), "cache_seqlens"),
    ("cache_write_fp8", dict(lens=Z(2)), "cache_seqlens"), ("cache_write_fp8", dict(k=Z(2, 1, 64, 2).half().transpose(2, 3)), "contiguous"),
    ("cache_write_fp8", dict(k=Z(2, 1, 2, 68).half()[..., :64]), "aligned"),
    ("cache_read_fp8", dict(out=torch.int8), "dtype"),
    ("window_attn_decode_fp8", dict(k=Z(2, 1, 4, 128).half()), "q must"), ("window_attn_decode_fp8", dict(k=Z(2, 1, 4, 64)), "float16 or"),
    ("window_attn_decode_fp8", dict(k=Z(2, 1, 3, 64).half()), "multiple"), ("window_attn_decode_fp8", dict(k=Z(2, 17, 2, 64).half()), "1 to 16"),
    ("window_attn_decode_fp8", dict(args=(0,)), "window"), ("window_attn_decode_fp8", dict(args=(5, -1)), "window"),
    ("window_attn_decode_fp8", dict(args=("a",)), "window"),
])
def test_cache_refusals(pkg, as_if_on_gpu, name, kw, match):
    with pytest.raises(ValueError, match=match):
        CALLS[name](pkg, {**_operands(), **kw})


@pytest.mark.parametrize("i", range(4))
def test_expanded_caches_are_not_written(pkg, as_if_on_gpu, i):
    """Two sequences (or heads) would write the same rows."""
    for dim in (0, 2):
        o = _operands()
        to = [o["kc"], o["kc"].clone(), o["ks"], o["ks"].clone()]
        to[i] = to[i].narrow(dim, 0, 1).expand_as(to[i])
        with pytest.raises(ValueError, match="expanded"):
            pkg.cache_write_fp8(o["k"], o["k"], *to, o["lens"])


@pytest.mark.parametrize("name,key", [("quantize_fp8", "y"), ("quantize_fp8_weight", "y"), ("fp8_linear", "xs"),
                                      ("fp8_linear", "ws"), ("cache_write_fp8", "k"), ("cache_read_fp8", "ks"),
                                      ("window_attn_decode_fp8", "k"), ("window_attn_decode_fp8", "ks")])
def test_no_gradient_is_refused(pkg, name, key):
    o = _operands()
    o[key] = o[key].clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="no gradient"):
        CALLS[name](pkg, o)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        CALLS[name](pkg, o)


@pytest.mark.parametrize("name,key", [("linear_xent", "x"), ("linear_xent", "w"), ("quantize_fp8", "y"), ("fp8_linear", "xs"),
                                      ("cache_write_fp8", "k"), ("window_attn_decode_fp8", "k")])
def test_forward_mode_is_refused(pkg, name, key):
    from torch.autograd import forward_ad
    for grad in (False, True):
        o = _operands()
        with forward_ad.dual_level():
            o[key] = forward_ad.make_dual(o[key].clone().requires_grad_(grad), torch.ones_like(o[key]))
            with pytest.raises(NotImplementedError, match="forward mode"):
                CALLS[name](pkg, o)


def test_scale_without_gradient_is_refused(pkg):
    s = torch.tensor(0.1, requires_grad=True)
    with pytest.raises(NotImplementedError, match="scale"):
        CALLS["window_attn_decode_fp8"](pkg, {**_operands(), "args": (None, 0, s)})


def test_sizes_beyond_32_bits(pkg):
    """Nothing is cut off on its way through the C boundary."""
    from importlib import import_module
    check = import_module("v100-attention-lab_amd.ops")._check_sizes
    check(0, 2 ** 31 - 1)
    with pytest.raises(ValueError, match="2\\^31"):
        check(5, 2 ** 31)
    L = import_module("v100-attention-lab_amd.loss")
    with pytest.raises(ValueError, match="2\\^31"):      # (checks before it pass on meta tensors)
        L._validate, keep = (lambda *a: None), L._validate
        try:
            L._plan(torch.empty(2 ** 31, 8, dtype=torch.float16, device="meta"), torch.empty(9, 8, dtype=torch.float16, device="meta"),
                    None, None, None, False)
        finally:
            L._validate = keep
