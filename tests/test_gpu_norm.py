"""GPU tests of add_rms_norm, add_rms_norm_bwd and add_rms_norm_fp8 against the
formulas in 64 bits.

Tolerances (2-norm of the difference over that of the result): sums and the
norm are held in fp32 (2^-19: a few roundings, and the tree sums of a row),
dweight's sum over rows adds one rounding a row of a workgroup in the worst
case (2^-17); a 16-bit output adds one rounding to its type."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -19
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


def _err(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.isfinite(got).all()
    n = want.norm()
    return ((got - want).norm() / n).item() if n > 0 else (got - want).norm().item()


def _inputs(dev, shape, xd, rd, wd, seed):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    D = shape[-1]
    return (rn(*shape).to(xd).to(dev), (2 * rn(*shape)).to(rd).to(dev), (1 + 0.3 * rn(D)).to(wd).to(dev),
            rn(*shape).to(xd).to(dev), rn(*shape).to(rd).to(dev))


def _norm(r, w, eps):
    rstd = 1 / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    return r * rstd * w, rstd


def _fwd_check(pkg, x, w, res, eps=1e-6):
    y, r = pkg.add_rms_norm(x, w, res, eps)
    torch.cuda.synchronize()
    s = x.double() + (res.double() if res is not None else 0.0)
    want, _ = _norm(s, w.double(), eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    if res is None:
        assert r is x
    else:
        assert r.dtype == res.dtype and _err(r, s) <= F32 + ROUND[r.dtype]
    assert _err(y, want) <= F32 + ROUND[y.dtype]
    return r


def _bwd_check(pkg, r, w, dy, dr, eps=1e-6):
    got, dw = pkg.add_rms_norm_bwd(r, w, dy, dr, eps)
    torch.cuda.synchronize()
    R, W, DY = r.double(), w.double(), dy.double()
    _, rstd = _norm(R, W, eps)
    n = R * rstd
    want = rstd * (W * DY - n * (W * DY * n).mean(-1, keepdim=True)) + (dr.double() if dr is not None else 0.0)
    assert got.dtype == r.dtype and dw.dtype == w.dtype
    # a row of one column has no gradient but dr: the two terms cancel
    size = max(want.norm().item(), (rstd * W * DY).norm().item())
    assert (got.double() - want).norm().item() <= (F32 + ROUND[got.dtype]) * size
    assert _err(dw, (DY * n).flatten(0, -2).sum(0)) <= 2.0 ** -17 + ROUND[dw.dtype]


@pytest.mark.parametrize("xd,rd", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (5, 64), (1, 512), (130, 520), (7, 1001), (9, 1024), (4, 2048),
                                    (3, 4096), (2, 4100), (5, 8192), (2, 16384), (3, 9001), (2, 16392), (700, 48)])
def test_forward_backward(pkg, cuda, xd, rd, rows, D):
    for wd in dict.fromkeys((xd, torch.float32)):
        x, res, w, dy, dr = _inputs(cuda, (rows, D), xd, rd, wd, seed=rows + D)
        r = _fwd_check(pkg, x, w, res)
        _fwd_check(pkg, x, w, None)
        _bwd_check(pkg, r, w, dy, dr)
        _bwd_check(pkg, r, w, dy, None)


@pytest.mark.parametrize("rows,D", [(1500, 520), (3000, 96), (1100, 4096), (1030, 1001), (600, 20000)])
def test_more_rows_than_partial_sums(pkg, cuda, rows, D):
    x, res, w, dy, dr = _inputs(cuda, (rows, D), torch.bfloat16, torch.float32, torch.float32, seed=1)
    _bwd_check(pkg, res, w, dy, dr)


def _fp8_check(pkg, x, w, res, group):
    y, scale, r = pkg.add_rms_norm_fp8(x, w, res, group=group)
    torch.cuda.synchronize()
    want, _ = _norm(x.double() + (res.double() if res is not None else 0.0), w.double(), 1e-6)
    D = x.shape[-1]
    assert y.dtype == torch.float8_e4m3fn and y.shape == x.shape
    assert scale.shape == (*x.shape[:-1], D // (group or D))
    top = want.unflatten(-1, (-1, group or D)).abs().amax(-1)
    s = scale.double().view(top.shape)
    assert ((s - top / 448).abs() <= 2.0 ** -18 * top / 448).all()
    back = (y.double().unflatten(-1, (-1, group or D)) * s[..., None]).flatten(-2)
    # e4m3: half a step is 2^-4 of the value, or 2^-10 of the scale below its normal range
    step = (2.0 ** -4 + 2.0 ** -16) * want.abs() + 2.0 ** -10 * 1.001 * s[..., None].expand(*s.shape, group or D).flatten(-2)
    assert ((back - want).abs() <= step).all()
    assert (y.float().abs() <= 448).all()


@pytest.mark.parametrize("xd,rd", TYPES)
@pytest.mark.parametrize("rows,D,group", [(1, 1, None), (5, 64, None), (3, 1001, None), (16, 2048, None),
                                          (16, 2048, 128), (3, 128, 128), (2, 4096, 128), (2, 8192, None),
                                          (3, 16512, 128), (2, 17000, None), (65, 384, 128)])
def test_fp8(pkg, cuda, xd, rd, rows, D, group):
    x, res, w, _, _ = _inputs(cuda, (rows, D), xd, rd, xd, seed=rows + D)
    _fp8_check(pkg, x, w, res, group)
    _fp8_check(pkg, x, w, None, group)


@pytest.mark.parametrize("rows,D", [(33, 64), (17, 72), (19, 128), (9, 136), (2100, 256), (5, 264), (13, 512), (6, 1016),
                                    (37, 63), (40, 65), (9, 101), (21, 133), (3, 255), (7, 257), (9000, 101), (5, 513)])
def test_rows_of_part_of_a_wave(pkg, cuda, rows, D):
    """Rows held by 8, 16 or 32 lanes, 8 columns and one column at a time."""
    for xd, rd in TYPES:
        x, res, w, dy, dr = _inputs(cuda, (rows, D), xd, rd, torch.float32, seed=rows + D)
        r = _fwd_check(pkg, x, w, res)
        _bwd_check(pkg, r, w, dy, dr)
        _fp8_check(pkg, x, w, res, None)
        if D % 128 == 0:
            _fp8_check(pkg, x, w, res, 128)


@pytest.mark.parametrize("group", [None, 128])
def test_fp8_misaligned(pkg, cuda, group):
    x, res, w, _, _ = _inputs(cuda, (6, 258), torch.bfloat16, torch.bfloat16, torch.float32, seed=2)
    _fp8_check(pkg, x[:, 1:257], w[1:257], res[:, 2:], group)


@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("xd", DTYPES)
def test_zero_and_tiny_rows(pkg, cuda, xd, group):
    """A row of zeros gives zeros with scale 0; a row far below eps keeps its
    precision (e4m3 of values scaled by 1 / sqrt(eps))."""
    x, _, w, dy, _ = _inputs(cuda, (4, 256), xd, xd, xd, seed=3)
    x[1] = 0
    x[2] = x[2] * 2.0 ** -14
    y, r = pkg.add_rms_norm(x, w)
    assert (y[1] == 0).all()
    q, s, _ = pkg.add_rms_norm_fp8(x, w, group=group)
    assert (q[1].float() == 0).all() and (s[1] == 0).all()
    _fwd_check(pkg, x, w, None)
    _fp8_check(pkg, x, w, None, group)
    _bwd_check(pkg, x, w, dy, None)


def test_fp8_smallest_scales(pkg, cuda):
    """Outputs so small that 448 / max leaves fp32 keep their ratios."""
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(1)).to(cuda)
    w = torch.full((128,), 2.0 ** -125, device=cuda)
    q, s, _ = pkg.add_rms_norm_fp8(x, w, eps=0.0)
    want = x / x.abs().amax(-1, keepdim=True) * 448
    assert ((q.float() - want).abs() <= 2.0 ** -3.9 * want.abs() + 2.0 ** -9).all()


def test_not_finite_rows_stay_apart(pkg, cuda):
    x, res, w, dy, dr = _inputs(cuda, (8, 512), torch.bfloat16, torch.bfloat16, torch.bfloat16, seed=4)
    clean = pkg.add_rms_norm(x, w, res)[0]
    clean_dr, _ = pkg.add_rms_norm_bwd(res, w, dy, dr)
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    y, r = pkg.add_rms_norm(x, w, res)
    keep = [0, 1, 2, 5, 6, 7]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all()
    for group in (None, 128):
        q, s, _ = pkg.add_rms_norm_fp8(x, w, res, group=group)
        assert torch.isnan(q[3].float()).all() and torch.isnan(s[3]).all() and torch.isfinite(s[keep]).all()
    res2 = res.clone()
    res2[2, 9] = float("nan")
    got, _ = pkg.add_rms_norm_bwd(res2, w, dy, dr)
    keep = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(got[keep], clean_dr[keep]) and torch.isnan(got[2]).all()


def test_shapes_and_strides(pkg, cuda):
    """[B, T, D] views, four leading dimensions, one row without any, no rows."""
    x, res, w, dy, dr = _inputs(cuda, (4, 6, 136), torch.float16, torch.float32, torch.float16, seed=6)
    cut = lambda t: t[1:3, ::2, 8:]
    for a, b, c, d, ww in ((cut(x), cut(res), cut(dy), cut(dr), w[8:].contiguous()),
                           (x.transpose(0, 1), res.transpose(0, 1), dy.transpose(0, 1), dr.transpose(0, 1), w),
                           (x[..., 1:], res[..., 1:], dy[..., 1:], dr[..., 1:], w[1:]),
                           (x.view(2, 2, 6, 136), res.view(2, 2, 6, 136), dy.view(2, 2, 6, 136), dr.view(2, 2, 6, 136), w),
                           (x.view(2, 2, 6, 136).transpose(0, 2), res.view(2, 2, 6, 136).transpose(0, 2),
                            dy.view(2, 2, 6, 136).transpose(0, 2), dr.view(2, 2, 6, 136).transpose(0, 2), w)):
        _fwd_check(pkg, a, ww, b)
        _bwd_check(pkg, b, ww, c, d)
    _fwd_check(pkg, x[0, 0], w, res[0, 0])
    y, r = pkg.add_rms_norm(x[:0], w, res[:0])
    assert y.shape == r.shape == (0, 6, 136)
    d0, dw = pkg.add_rms_norm_bwd(res[:0], w, dy[:0], dr[:0])
    assert d0.shape == (0, 6, 136) and (dw == 0).all()
    q, s, _ = pkg.add_rms_norm_fp8(x[:0], w, res[:0])
    assert q.shape == (0, 6, 136) and s.shape == (0, 6, 1)


@pytest.mark.parametrize("xd,rd", TYPES)
def test_autograd(pkg, cuda, xd, rd):
    x, res, w, dy, dr = _inputs(cuda, (2, 9, 264), xd, rd, xd, seed=7)
    a, b, c = (t.clone().requires_grad_() for t in (x, res, w))
    y, r = pkg.add_rms_norm(a, c, b)
    torch.autograd.backward([y, r], [dy, dr])
    want, dw = pkg.add_rms_norm_bwd(r.detach(), w, dy, dr)
    assert torch.equal(b.grad, want) and torch.equal(c.grad, dw)
    assert a.grad.dtype == xd and _err(a.grad, want) <= ROUND[xd] + 2.0 ** -20
    a2, c2 = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, r = pkg.add_rms_norm(a2, c2)
    y.backward(dy)
    want, dw = pkg.add_rms_norm_bwd(x, w, dy)
    assert torch.equal(a2.grad, want) and torch.equal(c2.grad, dw)


def test_gradient_and_differences(pkg, cuda):
    x, res, w, dy, dr = _inputs(cuda, (3, 72), torch.float32, torch.float32, torch.float32, seed=8)
    g, dw = pkg.add_rms_norm_bwd(x + res, w, dy, dr)
    f = lambda x, w: ((lambda o: (o[0].double() * dy).sum() + (o[1].double() * dr).sum())(pkg.add_rms_norm(x, w, res))).item()
    v, u = torch.randn(3, 72, device=cuda), torch.randn(72, device=cuda)
    eps = 2.0 ** -8
    dv = (f(x + eps * v, w) - f(x - eps * v, w)) / (2 * eps)
    du = (f(x, w + eps * u) - f(x, w - eps * u)) / (2 * eps)
    # eps^2 terms and fp32 roundings over eps
    assert abs(dv - (g.double() * v).sum().item()) <= 2.0 ** -10 * (g.norm() * v.norm()).item()
    assert abs(du - (dw.double() * u).sum().item()) <= 2.0 ** -10 * (dw.norm() * u.norm()).item()


def test_other_stream_and_repeat(pkg, cuda):
    x, res, w, dy, dr = _inputs(cuda, (2000, 512), torch.bfloat16, torch.float32, torch.bfloat16, seed=9)
    first = (*pkg.add_rms_norm(x, w, res), *pkg.add_rms_norm_bwd(res, w, dy, dr))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = (*pkg.add_rms_norm(x, w, res), *pkg.add_rms_norm_bwd(res, w, dy, dr))
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_eps_changed_in_place(pkg, cuda):
    """An eps that comes as a tensor counts by its value at the call, in the
    backward too."""
    gen = torch.Generator(device=cuda).manual_seed(71)
    x, dy = (torch.randn(6, 64, generator=gen, device=cuda) for _ in range(2))
    w = torch.ones(64, device=cuda)
    grads = []
    for change in (False, True):
        eps = torch.tensor(0.5)
        a = x.clone().requires_grad_()
        y, _ = pkg.add_rms_norm(a, w, None, eps)
        if change:
            eps.fill_(5.0)
        y.backward(dy)
        grads.append(a.grad)
    assert torch.equal(*grads)


def test_no_rows_of_many_dimensions(pkg, cuda):
    x = torch.zeros(2, 3, 0, 8, device=cuda)
    w = torch.ones(8, device=cuda)
    y, r = pkg.add_rms_norm(x, w, x)
    assert y.shape == r.shape == x.shape
    dr, dw = pkg.add_rms_norm_bwd(r, w, y)
    assert dr.shape == x.shape and (dw == 0).all()
    y, scale, _ = pkg.add_rms_norm_fp8(x, w)
    assert y.shape == x.shape and scale.shape == (2, 3, 0, 1)


def test_more_rows_than_a_launch_holds(pkg, cuda):
    """2^29 rows of 8 threads each are more than 32 bits of threads."""
    rows, D = 2 ** 29 + 3, 8
    gen = torch.Generator(device=cuda).manual_seed(81)
    row = torch.randn(1, D, generator=gen, device=cuda).to(torch.bfloat16)
    w = torch.randn(D, generator=gen, device=cuda).to(torch.bfloat16)
    y, r = pkg.add_rms_norm(row.expand(rows, D), w)
    want, _ = pkg.add_rms_norm(row, w)
    words, want = y.view(torch.int64), want.view(torch.int64)       # a row is two
    for i in range(0, rows, 2 ** 26):
        assert (words[i:i + 2 ** 26] == want).all(), i


@pytest.mark.parametrize("rows,D,group", [(700, 2048, None), (300, 4096, 128), (900, 1001, None), (50, 20000, None),
                                          (60, 16512, 128)])
def test_fp8_is_the_output_over_its_scale(pkg, cuda, rows, D, group):
    """fp32 rows: the bytes are the 32-bit output divided by the scale that is
    returned, rounded to the nearest (ties to even), bit for bit."""
    x, res, w, _, _ = _inputs(cuda, (rows, D), torch.float32, torch.float32, torch.float32, seed=rows)
    y, _ = pkg.add_rms_norm(x, w, res)
    q, s, _ = pkg.add_rms_norm_fp8(x, w, res, group=group)
    want = (y.unflatten(-1, (-1, group or D)) / s[..., None]).flatten(-2).clamp(-448, 448).cpu().to(torch.float8_e4m3fn)
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))
