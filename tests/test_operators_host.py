"""CPU tests of the scan, norm and attention calls: the ctypes mirrors against
the header, the refusals of the C ABI (nothing is enqueued) and of the Python
surface, and the workspace sizes."""

import ctypes
import os
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(REPO, "include")
FAKE = 0x100000       # never read: every refusal below comes before the launch


@pytest.fixture(scope="module")
def lib(pkg):
    if not os.path.exists(pkg.LIB_PATH):
        from importlib import import_module
        import_module("v100-attention-lab_amd.build").build(verbose=False)
    return pkg.load_library()


@pytest.mark.parametrize("struct", ["GdnScanParams", "GdnNormParams", "GdnAttnParams", "GdnAttnDecodeParams"])
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


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------

def _scan(L, **kw):
    P = L.GdnScanParams()
    P.x = P.g = P.y = P.final_state = P.dy = P.dx = P.dg = P.workspace = FAKE
    P.workspace_bytes = 1 << 40
    P.B, P.T, P.D, P.N = 2, 1000, 256, 2
    P.x_dtype, P.g_dtype = L.DTYPE_BF16, L.DTYPE_F32
    for k, v in kw.items():
        setattr(P, k, v)
    return P


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), 1001), (dict(g=None), 1001), (dict(y=None), 1001), (dict(final_state=None), 1001),
    (dict(B=0), 1002), (dict(T=-1), 1002), (dict(D=0), 1002), (dict(N=3), 1002), (dict(cu_seqlens=FAKE), 1002),
    (dict(D=1 << 30, T=1 << 20), 1002), (dict(x_dtype=7), 1005), (dict(g_dtype=1), 1005),
    (dict(workspace=None), 1006), (dict(workspace=FAKE + 16), 1006), (dict(workspace_bytes=100), 1006)])
def test_scan_refusals(lib, pkg, kw, code):
    assert lib.gdn_scan_launch(ctypes.byref(_scan(pkg._lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", [(dict(dy=None), 1001), (dict(dx=None), 1001), (dict(dg=None), 1001),
                                     (dict(D=-1), 1002), (dict(workspace_bytes=0), 1006)])
def test_scan_bwd_refusals(lib, pkg, kw, code):
    assert lib.gdn_scan_bwd_launch(ctypes.byref(_scan(pkg._lib, **kw)), None) == code


def test_scan_sizes(lib, pkg):
    size = lambda **kw: lib.gdn_scan_workspace_size(ctypes.byref(_scan(pkg._lib, **kw)))
    bwd = lambda **kw: lib.gdn_scan_bwd_workspace_size(ctypes.byref(_scan(pkg._lib, **kw)))
    C = lib.gdn_scan_chunk()
    assert lib.gdn_scan_slots(2, 1000, 2, 0) == 2 * -(-1000 // C)
    assert lib.gdn_scan_slots(1, 1000, 5, 1) == 1000 // C + 5
    assert lib.gdn_scan_slots(0, 10, 1, 0) == -1
    assert size(T=C) == 0 and size(T=0) == 0 and bwd(T=C) == 0     # one chunk a sequence
    pairs = 2 * -(-1000 // C) * 256 * 8
    assert pairs <= size() <= pairs * 17 // 16 + 1024
    assert bwd() == size() + 2 * -(-1000 // C) * 256 * 4           # and the states
    assert bwd(states=FAKE) == size()
    assert size(D=0) == -1 and lib.gdn_scan_workspace_size(None) == -1
    assert lib.gdn_scan_launch(None, None) == 1001 and lib.gdn_scan_bwd_launch(None, None) == 1001


def _norm(L, **kw):
    P = L.GdnNormParams()
    for n in ("x", "res", "w", "y", "r_out", "r", "dy", "dr", "dw", "workspace"):
        setattr(P, n, FAKE)
    P.workspace_bytes = 1 << 40
    P.n_outer, P.n_inner, P.D, P.eps = 1, 10, 256, 1e-6
    P.x_dtype, P.r_dtype, P.w_dtype = L.DTYPE_BF16, L.DTYPE_F32, L.DTYPE_BF16
    for k, v in kw.items():
        setattr(P, k, v)
    return P


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), 1001), (dict(w=None), 1001), (dict(y=None), 1001), (dict(r_out=None), 1001),
    (dict(D=0), 1002), (dict(n_outer=-1), 1002), (dict(n_outer=1 << 20, n_inner=1 << 20), 1002),
    (dict(group=64, scale=FAKE), 1003), (dict(group=128), 1003), (dict(group=128, scale=FAKE, D=200), 1003),
    (dict(x_dtype=9), 1005), (dict(r_dtype=1), 1005), (dict(w_dtype=1), 1005), (dict(res=None), 1005)])
def test_norm_refusals(lib, pkg, kw, code):
    assert lib.gdn_norm_launch(ctypes.byref(_norm(pkg._lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(r=None), 1001), (dict(dy=None), 1001), (dict(dr=None), 1001), (dict(dw=None), 1001), (dict(D=-4), 1002),
    (dict(w_dtype=5), 1005), (dict(workspace=None), 1006), (dict(workspace_bytes=64), 1006)])
def test_norm_bwd_refusals(lib, pkg, kw, code):
    assert lib.gdn_norm_bwd_launch(ctypes.byref(_norm(pkg._lib, **kw)), None) == code


def test_norm_no_rows_is_nothing(lib, pkg):
    assert lib.gdn_norm_launch(ctypes.byref(_norm(pkg._lib, n_inner=0)), None) == 0
    assert lib.gdn_norm_launch(None, None) == 1001


def _attn(L, **kw):
    P = L.GdnAttnParams()
    for n in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "workspace"):
        setattr(P, n, FAKE)
    P.workspace_bytes = 1 << 40
    P.B, P.Tq, P.Tk, P.N, P.Hq, P.Hk, P.D, P.window, P.sinks, P.scale = 2, 100, 100, 2, 4, 2, 64, 50, 2, 0.1
    for n, h in (("q", 4), ("o", 4), ("do", 4), ("dq", 4), ("k", 2), ("v", 2), ("dk", 2), ("dv", 2)):
        getattr(P, f"{n}_stride")[:] = (100 * h * 64, h * 64, 64)
    P.dtype = L.DTYPE_F16
    for k, v in kw.items():
        if k.endswith("_stride"):
            getattr(P, k)[:] = v
        else:
            setattr(P, k, v)
    return P


ATTN_COMMON = [
    (dict(q=None), 1001), (dict(k=None), 1001), (dict(o=None), 1001), (dict(B=0), 1002), (dict(Tq=-1), 1002),
    (dict(Hq=5), 1002), (dict(Hk=0), 1002), (dict(N=1), 1002), (dict(cu_seqlens=FAKE, B=2), 1002),
    (dict(cu_seqlens=FAKE, B=1, Tk=99), 1002), (dict(window=0), 1002), (dict(sinks=-1), 1002),
    (dict(Tq=1 << 30, Tk=1 << 30), 1002), (dict(D=96), 1003), (dict(D=256), 1003), (dict(dtype=0), 1005),
    (dict(q=FAKE + 8), 1004), (dict(k_stride=(6400, 132, 64)), 1004), (dict(v=FAKE + 2), 1004)]


@pytest.mark.parametrize("kw,code", ATTN_COMMON)
def test_attn_refusals(lib, pkg, kw, code):
    assert lib.gdn_attn_launch(ctypes.byref(_attn(pkg._lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", ATTN_COMMON + [
    (dict(lse=None), 1001), (dict(d_o=None), 1001), (dict(dq=None), 1001), (dict(dv=None), 1001),
    (dict(d_o=FAKE + 4), 1004), (dict(dk_stride=(6400, 130, 64)), 1004), (dict(workspace=None), 1006),
    (dict(workspace=FAKE + 8), 1006), (dict(workspace_bytes=1000), 1006)])
def test_attn_bwd_refusals(lib, pkg, kw, code):
    assert lib.gdn_attn_bwd_launch(ctypes.byref(_attn(pkg._lib, **kw)), None) == code


def test_attn_nothing_to_do_and_sizes(lib, pkg):
    L = pkg._lib
    assert lib.gdn_attn_launch(ctypes.byref(_attn(L, Tq=0)), None) == 0
    assert lib.gdn_attn_launch(None, None) == 1001 and lib.gdn_attn_bwd_launch(None, None) == 1001
    size = lambda **kw: lib.gdn_attn_bwd_workspace_size(ctypes.byref(_attn(L, **kw)))
    assert size(D=96) == -1 and lib.gdn_attn_bwd_workspace_size(None) == -1
    # lse and D of every row; parts of the first keys stay below the rows' own size in fp32, several times
    rows = 4 * 20000 * 16
    big = dict(B=4, N=4, Tq=20000, Tk=20000, Hq=16, Hk=4, D=128, window=1024, dtype=L.DTYPE_BF16)
    assert rows * 8 <= size(sinks=0, **big) < rows * 8 + 4096
    assert size(sinks=4, **big) < rows * 8 + 3 * 4 * 20000 * 4 * 128 * 8


def _decode(L, **kw):
    P = L.GdnAttnDecodeParams()
    for n in ("q", "k", "v", "o", "cache_seqlens", "workspace"):
        setattr(P, n, FAKE)
    P.workspace_bytes = 1 << 40
    P.B, P.T, P.S, P.Hq, P.Hk, P.D, P.window, P.sinks, P.scale = 2, 1, 4096, 8, 2, 128, 4096, 0, 0.1
    P.q_stride[:] = P.o_stride[:] = (8 * 128, 8 * 128, 128)
    P.k_stride[:] = P.v_stride[:] = (4096 * 256, 256, 128)
    P.dtype = L.DTYPE_BF16
    for k, v in kw.items():
        if k.endswith("_stride"):
            getattr(P, k)[:] = v
        else:
            setattr(P, k, v)
    return P


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1001), (dict(cache_seqlens=None), 1001), (dict(o=None), 1001), (dict(T=0), 1002), (dict(T=17), 1002),
    (dict(S=0), 1002), (dict(Hq=7), 1002), (dict(window=0), 1002), (dict(sinks=-2), 1002), (dict(D=80), 1003),
    (dict(dtype=0), 1005), (dict(k=FAKE + 8), 1004), (dict(v_stride=(4096 * 256, 260, 128)), 1004),
    (dict(workspace=None), 1006), (dict(workspace_bytes=16), 1006)])
def test_decode_refusals(lib, pkg, kw, code):
    assert lib.gdn_attn_decode_launch(ctypes.byref(_decode(pkg._lib, **kw)), None) == code


def test_attn_workspace_of_few_rows(lib, pkg):
    """Parts (a maximum, a sum and D values a row and split) only where few blocks
    of rows share long keys, at most 512 blocks of them."""
    size = lambda **kw: lib.gdn_attn_workspace_size(ctypes.byref(_attn(pkg._lib, **kw)))
    few = dict(Tq=40, Tk=5000, window=5000)
    assert size() == 0 and size(Tq=40, Tk=5000) == 0           # 100 keys; a short window
    assert 0 < size(**few) <= 512 * 128 * (64 + 2) * 4 + 256
    assert size(B=64, N=64, **few) == 0                        # enough blocks
    assert size(cu_seqlens=FAKE, B=1, Tq=5000, Tk=5000, window=5000) == 0
    assert size(D=96) == -1 and lib.gdn_attn_workspace_size(None) == -1
    for kw in (dict(workspace=None), dict(workspace_bytes=100), dict(workspace=FAKE + 16)):
        assert lib.gdn_attn_launch(ctypes.byref(_attn(pkg._lib, **few, **kw)), None) == 1006


def test_decode_workspace(lib, pkg):
    size = lambda **kw: lib.gdn_attn_decode_workspace_size(ctypes.byref(_decode(pkg._lib, **kw)))
    assert size() > 0 and size(B=512) == 0          # enough sequences: no splits, no parts
    assert size(D=80) == -1 and lib.gdn_attn_decode_workspace_size(None) == -1


def test_status_texts(pkg):
    for code in (1001, 1002, 1003, 1004, 1005, 1006):
        assert "gdn_fwd" not in pkg._lib.op_status_string(code)
    assert pkg._lib.op_status_string(1) != ""


# ---------------------------------------------------------------------------
# Python surface (everything here is refused before the device matters)
# ---------------------------------------------------------------------------

def test_cpu_tensors_are_refused(pkg):
    x = torch.zeros(1, 4, 8)
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    lens = torch.ones(1, dtype=torch.int32)
    for call in (lambda: pkg.gated_scan(x, x), lambda: pkg.gated_scan_bwd(x, x, None, x),
                 lambda: pkg.add_rms_norm(x, x[0, 0]), lambda: pkg.add_rms_norm_fp8(x, x[0, 0]),
                 lambda: pkg.add_rms_norm_bwd(x, x[0, 0], x), lambda: pkg.window_attn(q, q, q),
                 lambda: pkg.window_attn_bwd(q, q, q, q, torch.zeros(1, 4, 2), q),
                 lambda: pkg.window_attn_decode(q, q, q, lens)):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("args,kw,msg", [
    ((torch.zeros(4, 8), torch.zeros(4, 8)), {}, r"\[B, T, D\]"),
    (("x", "g"), {}, r"\[B, T, D\]"),
    ((torch.zeros(1, 4, 8), torch.zeros(1, 4, 9)), {}, "g must be"),
    ((torch.zeros(1, 4, 8, dtype=torch.float64), torch.zeros(1, 4, 8)), {}, "dtype"),
    ((torch.zeros(1, 4, 8), torch.zeros(1, 4, 8).half()), {}, "g must be float32"),
    ((torch.zeros(1, 4, 0), torch.zeros(1, 4, 0)), {}, "positive"),
    ((torch.zeros(1, 4, 8), torch.zeros(1, 4, 8), torch.zeros(2, 8)), {}, "h0"),
    ((torch.zeros(1, 4, 8), torch.zeros(1, 4, 8), torch.zeros(1, 8).half()), {}, "h0"),
    ((torch.zeros(2, 4, 8), torch.zeros(2, 4, 8)), {"cu_seqlens": torch.tensor([0, 4])}, "packed batch"),
    ((torch.zeros(1, 4, 8), torch.zeros(1, 4, 8)), {"cu_seqlens": torch.tensor([0.0, 4.0])}, "int64"),
    ((torch.zeros(1, 4, 8), torch.zeros(1, 4, 8)), {"cu_seqlens": [0, 4]}, "1-D"),
])
def test_scan_arguments(pkg, args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        pkg.gated_scan(*args, **kw)


@pytest.mark.parametrize("change,msg", [
    (dict(k=torch.zeros(1, 4, 2, 128, dtype=torch.float16)), "must be"),
    (dict(v=torch.zeros(1, 5, 2, 64, dtype=torch.float16)), "must be"),
    (dict(k=torch.zeros(1, 4, 3, 64, dtype=torch.float16), v=torch.zeros(1, 4, 3, 64, dtype=torch.float16)), "multiple"),
    (dict(q=torch.zeros(1, 4, 4, 64)), "float16 or bfloat16"),
    (dict(q=torch.zeros(1, 4, 4, 96, dtype=torch.float16), k=torch.zeros(1, 4, 2, 96, dtype=torch.float16),
          v=torch.zeros(1, 4, 2, 96, dtype=torch.float16)), "D=96"),
    (dict(q=torch.zeros(4, 4, 64, dtype=torch.float16)), r"\[B, T, Hq, D\]"),
    (dict(window=0), "window"), (dict(window=2.5), "window"), (dict(sinks=-1), "sinks"),
])
def test_attn_arguments(pkg, change, msg):
    z = lambda h: torch.zeros(1, 4, h, 64, dtype=torch.float16)
    args = dict(q=z(4), k=z(2), v=z(2), window=3, sinks=0)
    args.update(change)
    with pytest.raises(ValueError, match=msg):
        pkg.window_attn(**args)


def test_decode_and_fp8_refuse_gradients(pkg):
    q = torch.zeros(1, 1, 2, 64, dtype=torch.float16, requires_grad=True)
    with pytest.raises(NotImplementedError, match="window_attn"):
        pkg.window_attn_decode(q, q, q, torch.ones(1, dtype=torch.int32))
    x = torch.zeros(2, 8, requires_grad=True)
    with pytest.raises(NotImplementedError, match="add_rms_norm"):
        pkg.add_rms_norm_fp8(x, torch.ones(8))


@pytest.mark.parametrize("args,msg", [
    ((torch.tensor(1.0), torch.ones(1)), "must be a"),
    ((torch.zeros(2, 8), torch.ones(7)), "weight"),
    ((torch.zeros(2, 8, dtype=torch.int32), torch.ones(8)), "dtype"),
    ((torch.zeros(2, 8), torch.ones(8), torch.zeros(2, 9)), "residual"),
    (("x", torch.ones(8)), "must be a"),
])
def test_norm_arguments(pkg, args, msg):
    with pytest.raises(ValueError, match=msg):
        pkg.add_rms_norm(*args)


@pytest.mark.parametrize("window", [1, 60, 128, 1000])
@pytest.mark.parametrize("sinks", [1, 4, 130])
def test_attn_bwd_parts_of_the_first_rows(lib, pkg, window, sinks):
    """The first block of 128 keys is in its window's reach of the positions up to
    window + 126; from the next on its sinks' gradients have parts."""
    def size(S, sinks, **kw):
        kw = dict(dict(B=1, N=1, Tq=S, Tk=S, window=window, sinks=sinks, Hq=64, Hk=64, dtype=pkg._lib.DTYPE_BF16), **kw)
        return lib.gdn_attn_bwd_workspace_size(ctypes.byref(_attn(pkg._lib, **kw)))
    for S in range(window + 100, window + 160):
        for kw in (dict(), dict(Tq=7), dict(cu_seqlens=FAKE)):
            # (64 key heads of 3 blocks and more: one workgroup a block)
            if 64 * -(-S // 128) >= 128:
                assert (size(S, sinks, **kw) > size(S, 0, **kw)) == (S >= window + 128), (S, kw)


def test_attn_bwd_workspace_of_many_sequences(lib, pkg):
    """Parts of the first keys only for sequences longer than the window and a
    block: their number follows from the rows, not from the sequences."""
    def size(N, sinks):
        kw = dict(cu_seqlens=FAKE, B=1, N=N, Tq=65536, Tk=65536, Hq=32, Hk=8, D=128, window=1024, sinks=sinks,
                  dtype=pkg._lib.DTYPE_BF16)
        return lib.gdn_attn_bwd_workspace_size(ctypes.byref(_attn(pkg._lib, **kw)))
    assert size(8, 4) <= size(56, 4) == size(2048, 4) <= 512 << 20      # 56 * 1152 rows are the most
    assert size(2048, 0) < 17 << 20


@pytest.mark.parametrize("shape", [(2, 3, 0, 8), (0, 2, 4, 8), (2, 0, 0, 8), (3, 2, 4, 0)])
def test_norm_no_rows_of_many_dimensions(pkg, shape):
    """Leading dimensions without rows are joined like others (the refusal here is
    of the CPU, or of rows without columns)."""
    x, w = torch.zeros(shape), torch.ones(shape[-1])
    msg = "GPU" if shape[-1] else "must be a"
    for call in (lambda: pkg.add_rms_norm(x, w), lambda: pkg.add_rms_norm(x, w, x), lambda: pkg.add_rms_norm_fp8(x, w),
                 lambda: pkg.add_rms_norm_bwd(x, w, x)):
        with pytest.raises(ValueError, match=msg):
            call()


def _once(pkg, monkeypatch, name):
    """(call, inputs): a differentiable operator with its two launches replaced by
    results of the right shapes."""
    mod = {"gdn_fwd": pkg.ops, "gated_scan": pkg.scan, "window_attn": pkg.attn, "add_rms_norm": pkg.norm}[name]
    x = torch.randn(1, 4, 8)
    q = torch.randn(1, 4, 2, 64)
    gate = torch.randn(1, 4, 2)
    case = {
        "gdn_fwd": ((q, q, q, gate, gate), lambda *a: (torch.ones_like(q), torch.ones(1, 2, 64, 64)),
                    lambda *a: (torch.ones_like(q),) * 3 + (torch.ones_like(gate),) * 2 + (None,)),
        "gated_scan": ((x, x), lambda *a: (torch.ones_like(x), torch.ones(1, 8), torch.ones(1, 8)),
                       lambda *a: (torch.ones_like(x), torch.ones_like(x), None)),
        "window_attn": ((q, q, q), lambda *a: (torch.ones_like(q), torch.ones(1, 4, 2)),
                        lambda *a: (torch.ones_like(q),) * 3),
        "add_rms_norm": ((x, torch.ones(8)), lambda *a: (torch.ones_like(x), None, a[0]),      # (r is x)
                         lambda *a: (torch.ones_like(x), None, torch.ones(8))),
    }
    inputs, fwd, bwd = case[name]
    monkeypatch.setattr(mod, "_run", fwd)
    monkeypatch.setattr(mod, "_run_bwd", bwd)
    return getattr(pkg, name), [t.clone().requires_grad_() for t in inputs]


@pytest.mark.parametrize("name", ["gdn_fwd", "gated_scan", "window_attn", "add_rms_norm"])
def test_second_derivatives_are_refused(pkg, monkeypatch, name):
    """The kernels' gradients have no graph: a gradient of theirs raises instead
    of leaving out its terms."""
    call, inputs = _once(pkg, monkeypatch, name)
    out = call(*inputs)
    out = out[0] if isinstance(out, tuple) else out
    grad, = torch.autograd.grad(out.sum(), inputs[0], create_graph=True)
    assert grad.requires_grad
    with pytest.raises(RuntimeError, match="second derivatives"):
        grad.square().sum().backward()
    call(*inputs)
    out = call(*inputs)
    (out[0] if isinstance(out, tuple) else out).sum().backward()       # first ones as before
    assert inputs[0].grad is not None


def _calls(pkg):
    x, w = torch.randn(1, 4, 64), torch.ones(64)
    q, gate = torch.randn(1, 4, 2, 64).half(), torch.randn(1, 4, 2)
    lens = torch.ones(1, dtype=torch.int32)
    return {
        "gdn_fwd": (pkg.gdn_fwd, (q, q, q, gate, gate)), "gdn_chunk_fwd": (pkg.gdn_chunk_fwd, (q, q, q, gate, gate)),
        "chunk_gated_delta_rule": (pkg.chunk_gated_delta_rule, (q, q, q, gate, gate)),
        "gated_scan": (pkg.gated_scan, (x, x)), "window_attn": (pkg.window_attn, (q, q, q)),
        "window_attn_decode": (pkg.window_attn_decode, (q, q, q, lens)),
        "add_rms_norm": (pkg.add_rms_norm, (x, w, x)), "add_rms_norm_fp8": (pkg.add_rms_norm_fp8, (x, w, x)),
    }


@pytest.mark.parametrize("name", ["gdn_fwd", "gdn_chunk_fwd", "chunk_gated_delta_rule", "gated_scan", "window_attn",
                                  "window_attn_decode", "add_rms_norm", "add_rms_norm_fp8"])
def test_forward_mode_is_refused(pkg, name):
    """Dual tensors: an error instead of a result without its tangent, whether or
    not they require grad."""
    from torch.autograd import forward_ad
    call, args = _calls(pkg)[name]
    for i in range(2):
        for grad in (False, True):
            with forward_ad.dual_level():
                dual = list(args)
                dual[i] = forward_ad.make_dual(args[i].clone().requires_grad_(grad), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward mode"):
                    call(*dual)
                with pytest.raises(ValueError, match="GPU"):        # other tensors beside it pass on
                    call(*args)


def test_scale_without_gradient_is_refused(pkg):
    """A scale that requires grad would get none."""
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    s = torch.tensor(0.1, requires_grad=True)
    lens = torch.ones(1, dtype=torch.int32)
    for call in (lambda: pkg.window_attn(q, q, q, scale=s), lambda: pkg.window_attn_decode(q, q, q, lens, scale=s)):
        with pytest.raises(NotImplementedError, match="scale"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="GPU"):
        pkg.window_attn(q, q, q, scale=s.detach())


def test_inline_assembly_names_m0():
    """Assembly that sets m0 says so to the compiler."""
    import glob
    import re
    found = 0
    for path in glob.glob(os.path.join(REPO, "v100-attention-lab_amd", "csrc", "*")):
        with open(path) as f:
            for asm in re.findall(r"asm volatile\((.*?)\);", f.read(), re.S):
                if re.search(r"_b32 m0,", asm):
                    found += 1
                    assert '"m0"' in asm.split("::")[1], (path, asm)
    assert found >= 3


@pytest.mark.parametrize("name,make,kw", [
    ("gdn_scan_launch", _scan, dict(B=1 << 17, N=1 << 17, T=9, D=8192)),
    ("gdn_scan_launch", _scan, dict(B=1 << 23, N=1 << 23, T=2, D=1024)),
    ("gdn_scan_launch", _scan, dict(B=1, N=1 << 23, cu_seqlens=FAKE, T=100, D=64)),
    ("gdn_scan_launch", _scan, dict(B=1, N=1, T=1, D=2 ** 31 - 1)),
    ("gdn_scan_launch", _scan, dict(B=1, N=1, T=2 ** 31 - 1, D=1)),
    ("gdn_scan_bwd_launch", _scan, dict(B=1 << 20, N=1 << 20, T=2, D=2048)),
    ("gdn_norm_launch", _norm, dict(D=2 ** 31 - 1)),
    ("gdn_norm_bwd_launch", _norm, dict(D=1 << 28)),
    ("gdn_attn_launch", _attn, dict(B=1, cu_seqlens=FAKE, N=1 << 22, Tq=1 << 22, Tk=1 << 22, Hq=4, Hk=4)),
    ("gdn_attn_launch", _attn, dict(B=1 << 20, N=1 << 20, Tq=1, Tk=1, Hq=16, Hk=16)),
    ("gdn_attn_launch", _attn, dict(B=1 << 20, N=1 << 20, Hq=1 << 12, Hk=1 << 12)),
    ("gdn_attn_bwd_launch", _attn, dict(B=1, cu_seqlens=FAKE, N=1 << 21, Tq=1 << 21, Tk=1 << 21, Hq=8, Hk=8)),
    ("gdn_attn_bwd_launch", _attn, dict(B=1 << 20, N=1 << 20, Hq=1 << 12, Hk=1 << 12)),
    ("gdn_attn_decode_launch", _decode, dict(B=1 << 20, Hq=16, Hk=16)),
    ("gdn_attn_decode_launch", _decode, dict(B=1, Hq=1 << 28, Hk=1, T=16)),
])
def test_more_workgroups_than_a_launch_holds(lib, pkg, name, make, kw):
    """A launch counts its threads in 32 bits and runs what is left of more: such
    calls are refused before any kernel (the norm's forward takes several launches)."""
    P = make(pkg._lib, **dict(dict(workspace_bytes=1 << 62), **kw))
    assert getattr(lib, name)(ctypes.byref(P), None) == 1002


@pytest.mark.parametrize("name", ["gdn_fwd", "gated_scan", "window_attn", "add_rms_norm"])
def test_second_derivatives_are_refused_beside_others(pkg, monkeypatch, name):
    """The same where the engine is asked for some inputs alone, which other paths
    of the graph reach as well, and for the gradient that came in."""
    call, inputs = _once(pkg, monkeypatch, name)
    out = call(*inputs)
    out = out[0] if isinstance(out, tuple) else out
    weight = torch.ones_like(out, requires_grad=True)
    for want in (inputs[0], weight):
        loss = (out * weight).sum() + inputs[0].pow(3).sum()
        grad, = torch.autograd.grad(loss, inputs[0], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(grad.square().sum(), want, allow_unused=True)
