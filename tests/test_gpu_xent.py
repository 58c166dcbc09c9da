"""GPU tests of linear_xent and linear_xent_bwd against the formulas in 64 bits.

Tolerances: a logit is a sum of D products of 16-bit numbers in fp32, off by at
most D 2^-24 of the sum of their sizes; with the sums of exponentials the losses
are within 2^-15 (1 + |lse|) at the D and V below.  G is rounded once to the
operands' type before the sums that it enters and the gradients once behind
them, independently: within 1.5 of the type's unit (2-norm) of the result or,
where the terms cancel, of the root of the sum of their squares.  By the losses'
bound the probability p in G = dloss (p - [v = t]) is off by p 2^-15 (1 + |lse|),
which does not shrink where p - 1 does: these errors enter the same sums (V = 1 has
p - 1 = 0 and nothing but them).  fp16 results below 2^-14 have steps of 2^-24: n of
them are off by at most n^0.5 2^-25 however small they are."""

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]


def oracle(x, w, target, dloss):
    """(loss, lse, dx, dw, sizes); rows without a target take part in nothing."""
    x, w, V = x.double(), w.double(), w.shape[0]
    counts = (target >= 0) & (target < V)
    x = torch.where(counts[:, None], x, 0.0)
    t = torch.where(counts, target, 0).long()
    l = x @ w.T
    lse = torch.logsumexp(l, 1)
    rows = torch.arange(len(t), device=x.device)
    loss = torch.where(counts, lse - l[rows, t], 0.0)
    g = torch.exp(l - lse[:, None])
    d = torch.where(counts, dloss.double(), 0.0)[:, None]
    off = g * d * 2.0 ** -15 * (1 + lse.abs())[:, None]
    g[rows, t] -= 1.0
    g *= d
    sizes = []
    for f in (lambda z: z.square() @ w.square(), lambda z: z.square().T @ x.square()):
        sizes.append((f(g).sum().sqrt().item(), f(off).sum().sqrt().item()))
    return loss, torch.where(counts, lse, 0.0), g @ w, g.T @ x, sizes


def _close(got, want, units, size, name):
    assert torch.isfinite(got).all(), name
    d, (size, off) = (got.double() - want).norm().item(), size
    bound = units * UNIT[got.dtype] * max(want.norm().item(), size) + off + 1e-30
    if got.dtype == torch.float16:
        bound += got.numel() ** 0.5 * 2.0 ** -25
    assert d <= bound, (name, d / bound)


def _losses(loss, lse, want, want_lse):
    assert ((loss.double() - want).abs() <= 2.0 ** -15 * (1 + want_lse.abs())).all()
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -15 * (1 + want_lse.abs())).all()


def _inputs(dev, N, D, V, dtype, seed, std=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(N, D, generator=gen, device=dev).to(dtype)
    w = (torch.randn(V, D, generator=gen, device=dev) * std / D ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=gen, device=dev)
    dloss = (0.5 + torch.rand(N, generator=gen, device=dev)) / max(N, 1)
    return x, w, t, dloss


def _check(pkg, x, w, t, dloss):
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    want, want_lse, wx, ww, sizes = oracle(x, w, t, dloss)
    _losses(loss, lse, want, want_lse)
    _close(dx, wx, 1.5, sizes[0], "dx")
    _close(dw, ww, 1.5, sizes[1], "dw")
    counts = (t >= 0) & (t < w.shape[0])
    assert (loss[~counts] == 0).all() and (lse[~counts] == 0).all() and (dx[~counts] == 0).all()
    return loss, lse, dx, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,V", [
    (1, 8, 1), (1, 64, 2), (3, 72, 7), (17, 128, 300), (63, 200, 129), (64, 64, 1000), (65, 136, 257), (130, 1096, 1003),
    (200, 2048, 513), (257, 64, 4099), (300, 520, 33333), (1025, 256, 64), (1000, 1024, 5000), (2100, 64, 7000)])
def test_loss_and_gradients(pkg, cuda, dtype, N, D, V):
    x, w, t, dloss = _inputs(cuda, N, D, V, dtype, N + D + V)
    t[::7] = -100
    t[2::11] = V
    t[-1] = V - 1
    _check(pkg, x, w, t, dloss)


def test_big_tiles_and_several_pieces(pkg, cuda):
    """Tiles of 256 x 256 in every product, and a vocabulary of more than one piece."""
    x, w, t, dloss = _inputs(cuda, 9000, 1536, 9001, torch.bfloat16, 5)
    t[torch.rand(9000, device=cuda) < 0.3] = -1
    _check(pkg, x, w, t, dloss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_do_not_count_may_hold_anything(pkg, cuda, dtype):
    x, w, t, dloss = _inputs(cuda, 333, 192, 777, dtype, 1)
    t[5:90], t[200], t[300] = -100, 777, 1 << 40
    x[5], x[6], x[200], x[300] = float("nan"), float("inf"), -float("inf"), float("nan")
    dloss[5], dloss[300] = float("nan"), float("inf")
    _check(pkg, x, w, t, dloss)


def test_no_row_counts(pkg, cuda):
    x, w, t, dloss = _inputs(cuda, 70, 64, 100, torch.float16, 1)
    loss, lse, dx, dw = _check(pkg, x, w, torch.full_like(t, -100), dloss)
    assert (dw == 0).all()


def test_no_rows(pkg, cuda):
    x, w, t, dloss = _inputs(cuda, 0, 64, 100, torch.float16, 1)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    assert loss.shape == (0,) and dx.shape == (0, 64) and dw.shape == (100, 64) and (dw == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_leading_dimensions(pkg, cuda, dtype):
    """Rows inside wider ones, a padded batch, targets of 32 bits."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(4, 50, 320, generator=gen, device=cuda).to(dtype)[:, :, 64:256]
    w = (torch.randn(500, 400, generator=gen, device=cuda) * 0.1).to(dtype)[:, 8:200]
    t = torch.randint(-1, 500, (4, 50), generator=gen, device=cuda, dtype=torch.int32)
    dloss = torch.rand(4, 50, generator=gen, device=cuda)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    assert loss.shape == t.shape and dx.shape == x.shape and dw.shape == w.shape
    want, want_lse, wx, ww, sizes = oracle(x.reshape(-1, 192), w, t.reshape(-1), dloss.reshape(-1))
    _losses(loss.reshape(-1), lse.reshape(-1), want, want_lse)
    _close(dx.reshape(-1, 192), wx, 1.5, sizes[0], "dx")
    _close(dw, ww, 1.5, sizes[1], "dw")


def test_guard_rows_are_left(pkg, cuda):
    """Nothing is written beside the outputs: the calls' memory is cut out of a filled one."""
    x, w, t, dloss = _inputs(cuda, 129, 72, 131, torch.bfloat16, 9)
    lib, L = pkg.load_library(), pkg._lib
    import ctypes
    P = L.GdnXentParams()
    P.N, P.D, P.V, P.x_stride, P.w_stride, P.dtype = 129, 72, 131, 72, 72, L.DTYPE_BF16
    bufs = {n: torch.full((s + 512,), 7.0, dtype=d, device=cuda) for n, s, d in (
        ("loss", 129, torch.float32), ("lse", 129, torch.float32), ("dx", 129 * 72, torch.bfloat16),
        ("dw", 131 * 72, torch.bfloat16))}
    P.x, P.w, P.target, P.dloss, P.dloss_stride = x.data_ptr(), w.data_ptr(), t.data_ptr(), dloss.data_ptr(), 1
    for n, b in bufs.items():
        setattr(P, n, b[256:].data_ptr())
    for fn in ("xent", "xent_bwd"):
        n = getattr(lib, f"gdn_{fn}_workspace_size")(ctypes.byref(P))
        ws = torch.full((n + 1024,), 7, dtype=torch.uint8, device=cuda)
        P.workspace, P.workspace_bytes = ws[512:].data_ptr(), n
        assert getattr(lib, f"gdn_{fn}_launch")(ctypes.byref(P), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert (ws[:512] == 7).all() and (ws[512 + n:] == 7).all()
    for n, b in bufs.items():
        assert (b[:256] == 7).all() and (b[-256:] == 7).all(), n


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_gradients_of_a_mean(pkg, cuda, dtype):
    """Rows of very different weights: fp16's unit keeps those 2^-10 below the largest."""
    x, w, t, dloss = _inputs(cuda, 500, 256, 3000, dtype, 21)
    for f in (1e-7, 1.0, 1e5):
        d = dloss * f * torch.where(torch.arange(500, device=cuda) % 2 == 0, 1.0, 2.0 ** -10)
        _, lse = pkg.linear_xent(x, w, t, return_lse=True)
        if dtype == torch.float16:      # the outputs' own range
            w2, d2 = w, d / d.abs().max()
        else:
            w2, d2 = w, d
        dx, _ = pkg.linear_xent_bwd(x, w2, t, lse, d2)
        wx = oracle(x, w2, t, d2)[2]
        for part in (slice(0, None, 2), slice(1, None, 2)):
            g = dx[part].double()
            # fp16 outputs below 2^-14 have steps of 2^-24
            floor = 2.0 ** -25 * wx[part].numel() ** 0.5 if dtype == torch.float16 else 0.0
            assert (g - wx[part]).norm() <= 1.5 * UNIT[dtype] * wx[part].norm() + floor


def test_large_logits(pkg, cuda):
    """Sure predictions and logits of thousands: no exponential leaves its range."""
    x, w, t, dloss = _inputs(cuda, 200, 512, 900, torch.bfloat16, 4, std=400.0)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    want, want_lse, wx, ww, sizes = oracle(x, w, t, dloss)
    # logits of standard deviation 400 over sums of 512 terms of that size / 512^0.5
    assert ((lse.double() - want_lse).abs() <= 512 ** 0.5 * 400 * 2.0 ** -22).all()
    assert torch.isfinite(loss).all()
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_not_finite_rows_stay_their_own(pkg, cuda):
    x, w, t, dloss = _inputs(cuda, 100, 64, 500, torch.bfloat16, 4)
    x[3] = float("nan")
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    assert torch.isnan(loss[3]) and torch.isfinite(loss[torch.arange(100, device=cuda) != 3]).all()
    dx, _ = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    assert torch.isnan(dx[3]).all() and torch.isfinite(dx[torch.arange(100, device=cuda) != 3]).all()


def test_fixed_order(pkg, cuda):
    x, w, t, dloss = _inputs(cuda, 700, 512, 6000, torch.bfloat16, 8)
    runs = []
    for _ in range(3):
        loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
        runs.append((loss, lse, *pkg.linear_xent_bwd(x, w, t, lse, dloss)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


@pytest.mark.parametrize("reduction", ["sum", "mean", "weighted"])
def test_autograd(pkg, cuda, reduction):
    x, w, t, dloss = _inputs(cuda, 120, 96, 400, torch.bfloat16, 11)
    t[::5] = -100
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = pkg.linear_xent(xg.view(4, 30, 96), wg, t.view(4, 30))
    scale = {"sum": torch.ones_like(dloss), "mean": torch.full_like(dloss, 1 / 120), "weighted": dloss}[reduction]
    total = loss.sum() if reduction == "sum" else loss.mean() if reduction == "mean" else (loss.view(-1) * dloss).sum()
    total.backward()
    _, _, wx, ww, sizes = oracle(x, w, t, scale)
    _close(xg.grad, wx, 1.5, sizes[0], "dx")
    _close(wg.grad, ww, 1.5, sizes[1], "dw")


def test_gradient_against_differences(pkg, cuda):
    """(loss(x + h d) - loss(x - h d)) / 2h in 64 bits of the oracle's loss, d a
    direction, against the kernels' gradient along it."""
    x, w, t, _ = _inputs(cuda, 40, 64, 150, torch.bfloat16, 2)
    ones = torch.ones(40, device=cuda)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, ones)
    gen = torch.Generator(device=cuda).manual_seed(0)
    for at, grad in ((x, dx), (w, dw)):
        d = torch.randn(at.shape, generator=gen, device=cuda).double()
        h = 1e-4
        f = lambda s: oracle(*((at.double() + s * h * d, w) if at is x else (x, at.double() + s * h * d)), t, ones)[0].sum()
        want = (f(1) - f(-1)) / (2 * h)
        got = (grad.double() * d).sum()
        assert (got - want).abs() <= 1.5 * 2.0 ** -8 * grad.double().norm() * d.abs().max()


def test_second_derivative_raises(pkg, cuda):
    x, w, t, _ = _inputs(cuda, 10, 64, 50, torch.bfloat16, 2)
    x.requires_grad_()
    g, = torch.autograd.grad(pkg.linear_xent(x, w, t).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().square().sum().backward()


def test_captured_calls(pkg, cuda):
    """A captured step, replayed between eager calls on other inputs."""
    x, w, t, dloss = _inputs(cuda, 300, 128, 1000, torch.float16, 6)
    x2, w2, t2, d2 = _inputs(cuda, 300, 128, 1000, torch.float16, 7)

    def step():
        loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
        return (loss, lse, *pkg.linear_xent_bwd(x, w, t, lse, dloss))
    want = [r.clone() for r in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        pkg.linear_xent_bwd(x2, w2, t2, pkg.linear_xent(x2, w2, t2, return_lse=True)[1], d2)
    x.copy_(x2), w.copy_(w2), t.copy_(t2), dloss.copy_(d2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_another_stream(pkg, cuda):
    x, w, t, dloss = _inputs(cuda, 300, 128, 1000, torch.bfloat16, 6)
    want = pkg.linear_xent(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.linear_xent(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,V", [(5000, 64, 700), (3000, 8, 3000), (9000, 128, 9001), (700, 264, 40), (20000, 16, 7)])
def test_many_rows_of_few_columns(pkg, cuda, dtype, N, D, V):
    """Gradients whose tiles do not fill the card: the contraction in parts, of the
    weights' too (with a last piece of another size)."""
    x, w, t, dloss = _inputs(cuda, N, D, V, dtype, N + V)
    t[torch.rand(N, device=cuda) < 0.2] = -100
    _check(pkg, x, w, t, dloss)


def test_captured_autograd(pkg, cuda):
    """Forward and backward through autograd in one graph, the leaves made in it, while
    an eager graph of the same memory lives."""
    x, w, t, _ = _inputs(cuda, 200, 128, 700, torch.bfloat16, 6)

    def step():
        xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = pkg.linear_xent(xg, wg, t).sum()
        return (loss, *torch.autograd.grad(loss, (xg, wg)))
    want = [r.detach().clone() for r in step()]
    eager = pkg.linear_xent(x.detach().requires_grad_(), w, t).sum()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:])), i
        step()
    assert torch.isfinite(eager)


def test_one_gradient_alone(pkg, cuda):
    """x or the weight without a gradient, a weight that is expanded from one row."""
    x, w, t, _ = _inputs(cuda, 60, 64, 100, torch.bfloat16, 6)
    ones = torch.ones(60, device=cuda)
    _, _, wx, ww, sizes = oracle(x, w, t, ones)
    xg = x.clone().requires_grad_()
    pkg.linear_xent(xg, w, t).sum().backward()
    _close(xg.grad, wx, 1.5, sizes[0], "dx")
    wg = w.clone().requires_grad_()
    pkg.linear_xent(x, wg, t).sum().backward()
    _close(wg.grad, ww, 1.5, sizes[1], "dw")
    row = w[:1].clone().requires_grad_()
    pkg.linear_xent(x, row.expand(100, 64), t).sum().backward()
    # every word has the same logit: the gradient of their common weights is 0, of terms of this size
    g = torch.full((60, 100), 0.01, device=cuda, dtype=torch.float64)
    g[torch.arange(60, device=cuda), t] -= 1
    size = (g.abs().T @ x.double().abs()).sum(0).norm()
    assert row.grad.double().norm() <= 2 * 2.0 ** -8 * size


def test_offsets_beyond_32_bits(pkg, cuda):
    """A weight of more than 2^31 elements: the last words against the formulas."""
    V, D, N = 530_000, 4096, 20
    gen = torch.Generator(device=cuda).manual_seed(1)
    w = torch.empty(V, D, dtype=torch.bfloat16, device=cuda)
    for v in range(0, V, 100_000):
        w[v:v + 100_000] = torch.randn(min(100_000, V - v), D, generator=gen, device=cuda) * (2.0 / 64)
    x = torch.randn(N, D, generator=gen, device=cuda).bfloat16()
    t = torch.randint(V - 3000, V, (N,), generator=gen, device=cuda)
    dloss = torch.ones(N, device=cuda)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    logits = torch.cat([x.double() @ w[v:v + 50_000].double().T for v in range(0, V, 50_000)], 1)
    want_lse = torch.logsumexp(logits, 1)
    _losses(loss, lse, want_lse - logits[torch.arange(N, device=cuda), t], want_lse)
    p = torch.exp(logits - want_lse[:, None])
    g = p.clone()
    g[torch.arange(N, device=cuda), t] -= 1
    for part in (slice(0, 2000), slice(V - 4000, V)):
        _close(dw[part], g[:, part].T @ x.double(), 1.5, ((g[:, part].square().T @ x.double().square()).sum().sqrt().item(), 1e-3), "dw")
    want = sum(g[:, v:v + 50_000] @ w[v:v + 50_000].double() for v in range(0, V, 50_000))
    _close(dx, want, 1.5, (want.norm().item(), 0.0), "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["expanded", "rows", "padded"])
def test_a_mean_adds_no_error_of_its_own(pkg, cuda, dtype, form):
    """1 / 511 lies half a step of bf16 from its neighbours: G's largest terms, -dloss of
    every row, are not to be off by that.  Logits of 0 and 4096 words: p = 2^-12 within
    2^-11.8 of itself, and 1 - p is rounded to 1 in either type (2^-12 off at most); so an
    element of dx is off by the rounding of p (2^-11 of it, in fp16) over all words, by
    the target's 2^-12 and by its own half step."""
    N, D, V = 511, 64, 4096
    gen = torch.Generator(device=cuda).manual_seed(2)
    w = torch.randn(V, D, generator=gen, device=cuda).to(dtype)
    x = torch.zeros(N, D, device=cuda, dtype=dtype)
    t = torch.randint(0, V, (N,), generator=gen, device=cuda)
    dloss = torch.full((1,), 1 / 511, device=cuda).expand(N)
    if form != "expanded":
        dloss = dloss.contiguous()
    if form == "padded":
        t[::7], dloss[::7] = -100, 100.0
    _, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, _ = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    counts = (t >= 0)[:, None]
    W, Wt = w.double(), w.double()[t.clamp(min=0)]
    want = torch.where(counts, (W.mean(0) - Wt) * dloss.double()[:, None], 0.0)
    off = (Wt.abs() * (2.0 ** -12 + 2.0 ** -20) + W.abs().mean(0) * (2.0 ** -11 + 2.0 ** -11.8)) / 511
    bound = UNIT[dtype] * (want.abs() + off) + off + 2.0 ** -25
    assert ((dx.double() - want).abs() <= torch.where(counts, bound, 0.0)).all()
