"""GPU tests of fp8_linear, quantize_fp8 and quantize_fp8_weight.

Tolerances: products of e4m3 numbers are exact in fp32 and are summed there, at
most K + K / 128 additions and two roundings of a block's scales: a result is off
by at most (K + K / 128 + 3) 2^-24 of the sum of its terms' sizes, and by half a
step of its type.  16-bit results come from the 8-bit matrix unit, which cuts each
product at 2^-13 of the largest of its group of 8: every result is off by at most
8 2^-13 sum_groups largest <= 2^-10 of the sum of its terms' sizes more; and, the
cuts of terms of either sign being independent and evenly spread, their squares add
to 8 / 3 2^-26 sum_groups largest^2 <= 8 / 3 2^-26 sum terms^2, so that all results
together are within 2^-12 (2-norm) beside their rounding.  Quantised bytes are the quotient in fp32 rounded to the
nearest: within half a step of e4m3 (2^-4 of the value, 2^-10 near zero) and the
quotient's own rounding."""

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _bytes(shape, gen, dev):
    """e4m3 values of all sizes."""
    return (torch.randn(shape, generator=gen, device=dev) * torch.exp(torch.randn(shape, generator=gen, device=dev))).to(FP8)


def _operands(dev, M, K, N, seed, group=128):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x, w = _bytes((M, K), gen, dev), _bytes((N, K), gen, dev)
    xs = torch.exp(torch.randn(M, K // 128 if group else 1, generator=gen, device=dev))
    ws = torch.exp(torch.randn(-(-N // 128), K // 128, generator=gen, device=dev))
    return x, xs, w, ws


def oracle(x, xs, w, ws):
    """(y, sum of the terms' sizes) in 64 bits."""
    K, N = x.shape[1], w.shape[0]
    a = x.double() * xs.double().repeat_interleave(K // xs.shape[1], 1)
    b = w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
    return a @ b.T, a.abs() @ b.abs().T


def _check(y, want, size, K):
    assert torch.isfinite(y).all()
    off = (y.double() - want).abs()
    sums = (K + K // 128 + 3) * 2.0 ** -24 + (0.0 if y.dtype == torch.float32 else 2.0 ** -10)
    bound = sums * size * (1 + HALF[y.dtype]) + HALF[y.dtype] * want.abs() + \
        (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    assert (off <= bound).all(), (off / bound).max().item()
    if y.dtype != torch.float32 and y.numel() > 64:
        assert off.norm() <= (HALF[y.dtype] + 2.0 ** -12) * want.norm()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("M,K,N", [
    (1, 128, 1), (1, 2048, 2048), (3, 128, 17), (16, 1152, 131), (17, 256, 128), (31, 1280, 514), (33, 384, 1000),
    (64, 2304, 255), (65, 128, 64), (65, 512, 129), (100, 1024, 1003), (300, 768, 777), (513, 256, 2048),
    (1000, 640, 4097), (2100, 128, 3000), (4000, 384, 3900)])
@pytest.mark.parametrize("group", [128, 0])
def test_product(pkg, cuda, M, K, N, group, out):
    x, xs, w, ws = _operands(cuda, M, K, N, M + K + N, group)
    if out == torch.float16:        # its range
        xs, ws = xs / 64, ws / 64
    y = pkg.fp8_linear(x, xs, w, ws, out_dtype=out)
    assert y.shape == (M, N) and y.dtype == out
    _check(y, *oracle(x, xs, w, ws), K)


def test_rows_do_not_depend_on_others(pkg, cuda):
    """The same rows give the same bits in every batch that takes the same kernel,
    and NaN, infinite and zero scales stay in their own rows and columns."""
    x, xs, w, ws = _operands(cuda, 700, 512, 900, 4)
    y = pkg.fp8_linear(x, xs, w, ws)
    x2, xs2, ws2 = x.clone(), xs.clone(), ws.clone()
    x2.view(torch.uint8)[5, 300] = 0x7f       # NaN
    xs2[9, 1], xs2[11] = float("inf"), 0.0
    ws2[3, 2] = float("nan")
    z = pkg.fp8_linear(x2, xs2, w, ws2)
    assert torch.isnan(z[5]).all() and not torch.isfinite(z[9, :384]).any() and (z[11, :384] == 0).all()
    assert torch.isnan(z[:, 384:512]).all()
    keep = torch.tensor([i for i in range(700) if i not in (5, 9, 11)], device=cuda)
    cols = torch.tensor([i for i in range(900) if not 384 <= i < 512], device=cuda)
    assert torch.equal(z[keep][:, cols], y[keep][:, cols])


@pytest.mark.parametrize("M", [7, 200])
def test_strides_and_leading_dimensions(pkg, cuda, M):
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = _bytes((2, M, 1024), gen, cuda)[:, :, 256:640]
    w = _bytes((300, 512), gen, cuda)[:, 128:]
    xs = torch.rand(2, M, 6, generator=gen, device=cuda)[:, :, ::2]
    ws = torch.rand(3, 3, generator=gen, device=cuda)
    y = pkg.fp8_linear(x, xs, w, ws, out_dtype=torch.float32)
    assert y.shape == (2, M, 300)
    _check(y.view(-1, 300), *oracle(x.reshape(-1, 384), xs.reshape(-1, 3), w, ws), 384)
    z = pkg.fp8_linear(x[0, 0], xs[0, 0], w, ws, out_dtype=torch.float32)
    assert z.shape == (300,)
    _check(z[None], *oracle(x[0, :1], xs[0, :1], w, ws), 384)


def test_no_rows(pkg, cuda):
    x, xs, w, ws = _operands(cuda, 0, 256, 100, 1)
    assert pkg.fp8_linear(x, xs, w, ws).shape == (0, 100)
    q, s = pkg.quantize_fp8(torch.empty(0, 256, device=cuda))
    assert q.shape == (0, 256) and s.shape == (0, 2)


@pytest.mark.parametrize("M,N", [(5, 131), (40, 257), (129, 263)])
def test_guard_bytes_are_left(pkg, cuda, M, N):
    import ctypes
    x, xs, w, ws = _operands(cuda, M, 256, N, 1)
    L, lib = pkg._lib, pkg.load_library()
    buf = torch.full((M * N + 512,), 7.0, dtype=torch.bfloat16, device=cuda)
    P = L.GdnFp8LinearParams()
    P.x, P.x_scale, P.w, P.w_scale, P.y = (t.data_ptr() for t in (x, xs, w, ws, buf[256:]))
    P.x_stride, P.w_stride, P.M, P.N, P.K, P.group, P.y_dtype = 256, 256, M, N, 256, 128, L.DTYPE_BF16
    assert lib.gdn_fp8_linear_launch(ctypes.byref(P), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (buf[:256] == 7).all() and (buf[256 + M * N:] == 7).all()
    assert torch.equal(buf[256:256 + M * N].view(M, N), pkg.fp8_linear(x, xs, w, ws))


def _quant_oracle(x, group):
    """scale in fp32 as defined, and the quotients in 64 bits."""
    g = x.float().unflatten(-1, (-1, group))
    scale = (g.abs().amax(-1, keepdim=True).double() / 448.0).float()      # (a division by a number multiplies by its inverse)
    return scale.squeeze(-1), torch.where(scale > 0, g.double() / scale.double(), 0.0).flatten(-2)


def _quant_close(q, want):
    half = torch.clamp(want.abs() * 2.0 ** -4, min=2.0 ** -10)
    assert ((q.double() - want).abs() <= half * (1 + 2.0 ** -20) + want.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D", [(1, 128), (3, 384), (100, 2048), (33, 8320)])
@pytest.mark.parametrize("group", [128, None])
def test_quantize(pkg, cuda, dtype, M, D, group):
    gen = torch.Generator(device=cuda).manual_seed(M + D)
    x = (torch.randn(M, D, generator=gen, device=cuda) * torch.exp(3 * torch.randn(M, 1, generator=gen, device=cuda))).to(dtype)
    x[0, :128] = 0
    q, scale = pkg.quantize_fp8(x, group=group)
    want_scale, want = _quant_oracle(x, group or D)
    assert torch.equal(scale, want_scale)
    _quant_close(q, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", [(1, 128), (127, 256), (300, 384), (1024, 2048)])
def test_quantize_weight(pkg, cuda, dtype, N, K):
    gen = torch.Generator(device=cuda).manual_seed(N + K)
    w = (torch.randn(N, K, generator=gen, device=cuda) * 0.05).to(dtype)
    if N > 130:
        w[128:256, 128:256] = 0
    q, scale = pkg.quantize_fp8_weight(w)
    blocks = torch.nn.functional.pad(w.float(), (0, 0, 0, -N % 128)).view(-1, 128, K // 128, 128)
    want_scale = (blocks.abs().amax((1, 3)).double() / 448.0).float()
    assert torch.equal(scale, want_scale)
    full = want_scale.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
    _quant_close(q, torch.where(full > 0, w.double() / full, 0.0))


def test_quantize_not_finite(pkg, cuda):
    x = torch.randn(4, 256, device=cuda)
    x[1, 3], x[2, 200] = float("nan"), float("inf")
    q, s = pkg.quantize_fp8(x)
    assert torch.isnan(s[1, 0]) and torch.isnan(q[1, :128].float()).all() and torch.isfinite(q[1, 128:].float()).all()
    assert s[2, 1] == float("inf") and torch.isnan(q[2, 200].float()) and torch.isfinite(s[[0, 3]]).all()


def test_smallest_and_largest_values(pkg, cuda):
    """Scales near both ends of fp32's range."""
    for f in (1e-38, 1e-30, 1e30, 3e38):
        x = torch.linspace(-1, 1, 256, device=cuda).view(1, 256) * f
        q, s = pkg.quantize_fp8(x)
        want_scale, want = _quant_oracle(x, 128)
        assert torch.equal(s, want_scale)
        # a scale below the smallest normal number has few digits, but it is the one that counts
        _quant_close(q, want)


def test_norm_to_product(pkg, cuda):
    """The run of them together: the 8-bit norm's rows into a product, against the
    16-bit path; e4m3's half step 2^-4 on both operands' elements, independent."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(50, 1024, generator=gen, device=cuda).bfloat16()
    r = torch.randn(50, 1024, generator=gen, device=cuda)
    w = (torch.randn(1500, 1024, generator=gen, device=cuda) / 32).bfloat16()
    nw = torch.ones(1024, device=cuda)
    w8, ws = pkg.quantize_fp8_weight(w)
    for group in (128, None):
        y8, s, _ = pkg.add_rms_norm_fp8(x, nw, r, group=group)
        got = pkg.fp8_linear(y8, s, w8, ws, out_dtype=torch.float32)
        y, _ = pkg.add_rms_norm(x, nw, r)
        want = y.double() @ w.double().T
        assert ((got.double() - want).norm() / want.norm()) <= 2 ** 0.5 * 2.0 ** -4
        assert torch.equal(got, pkg.fp8_linear(y8, s, w8, ws, out_dtype=torch.float32))


def test_captured_calls(pkg, cuda):
    x = torch.randn(300, 512, device=cuda).bfloat16()
    w8, ws = pkg.quantize_fp8_weight(torch.randn(600, 512, device=cuda))
    run = lambda: pkg.fp8_linear(*pkg.quantize_fp8(x), w8, ws)
    want = run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run(), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for f in (1.0, -2.0, 0.5):
        x.mul_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, run())


@pytest.mark.parametrize("M,K,N", [(40_000, 128, 60_000), (17_000_000, 128, 24), (5, 128, 17_000_000)])
def test_offsets_beyond_32_bits(pkg, cuda, M, K, N):
    """Rows, weights or results of more than 2^31 bytes: the last ones against the formula."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    bytes_ = lambda n: torch.randint(0, 0x70, (n, K), generator=gen, device=cuda, dtype=torch.uint8).view(FP8)
    x, w = bytes_(M), bytes_(N)
    xs, ws = torch.rand(M, 1, generator=gen, device=cuda), torch.rand(-(-N // 128), 1, generator=gen, device=cuda)
    y = pkg.fp8_linear(x, xs, w, ws)
    m, n = min(M, 300), min(N, 300) // 4 * 4
    n0 = (N - n) // 128 * 128          # (whole blocks of outputs)
    for r in (slice(0, m), slice(M - m, M)):
        want, size = oracle(x[r], xs[r], w[n0:], ws[n0 // 128:])
        _check(y[r, n0:], want, size, K)


def test_quantize_beyond_32_bits(pkg, cuda):
    x = torch.zeros(9_000_000, 256, dtype=torch.bfloat16, device=cuda)
    x[-100:] = torch.randn(100, 256, device=cuda).bfloat16()
    for group in (128, None):
        q, s = pkg.quantize_fp8(x, group=group)
        q2, s2 = pkg.quantize_fp8(x[-100:].clone(), group=group)
        assert torch.equal(q[-100:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-100:], s2)
        assert (s[:-100] == 0).all()
