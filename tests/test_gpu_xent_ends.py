"""GPU tests of linear_xent at the ends of its range: sure predictions, logits of
thousands, dloss of every size and not finite, more logits than 2^37.

Where logits have to be exact, rows are unit vectors: the logits of row n are
column n % 64 of the weight, without a rounding."""

import math

import pytest
import torch
from test_gpu_xent import DTYPES, _close, _inputs, _losses, oracle

pytestmark = pytest.mark.gpu

D = 64
# every shape of the logits' tiles: 128 x 64, 128 x 128 in two forms, 256 x 256
SHAPES = [(48, 1000), (128, 2999), (1024, 8000), (1024, 10240)]


def _within(got, want, bound):
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1, worst


def _exact(dev, N, V, dtype, seed, std):
    """(x, w, t): logits w[:, n % 64], multiples of 1/64 cut to the type; a target a column."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.eye(D, device=dev).repeat(-(-N // D), 1)[:N].to(dtype)
    w = ((torch.randn(V, D, generator=gen, device=dev) * std * 64).round() / 64).to(dtype)
    t = torch.randperm(V, generator=gen, device=dev)[:D]
    return x, w, t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", SHAPES)
def test_sure_predictions(pkg, cuda, dtype, N, V):
    """Targets 18 to 40 above all others: no loss is below 0, and each is as far off as
    the sum of its exponentials, 1 and little more: at most 64 additions of a wave's
    lane, 1 of its halves, 2 of the waves, 2 tiles' of a thread of the join and 17 of its
    threads, half a unit of 2^-23 each, and as much for its logarithm.  The logarithm
    and its sum with the maximum's logit are rounded once each."""
    x, w, t = _exact(cuda, N, V, dtype, V, 3.0)
    cols = torch.arange(D, device=cuda)
    w[t, cols] = (w.float().amax(0) + torch.linspace(18, 40, D, device=cuda)).to(dtype)
    t = t[torch.arange(N, device=cuda) % D]
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    want, want_lse = oracle(x, w, t, torch.ones(N, device=cuda))[:2]
    assert loss.min().item() >= 0
    bound = 88 * 2.0 ** -24
    _within(loss, want, bound)
    _within(lse, want_lse, bound + 2.0 ** -24 * want_lse.abs())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", SHAPES)
def test_certain_predictions(pkg, cuda, dtype, N, V):
    """All other words 60 or more below: e^-60 V vanishes beside 1, so the loss is 0, lse
    the logit and the target's G 0, to the bit; the others' G sum to e^-60 V.  With a
    second word as large as the target the loss is ln 2, rounded once."""
    x, w, t = _exact(cuda, N, V, dtype, V, 3.0)
    cols, rows = torch.arange(D, device=cuda), torch.arange(N, device=cuda)
    w[t, cols] = (w.float().amax(0) + torch.linspace(60, 90, D, device=cuda)).to(dtype)
    top = w[t, cols].float()
    target = t[rows % D]
    loss, lse = pkg.linear_xent(x, w, target, return_lse=True)
    assert loss.abs().max().item() == 0 and torch.equal(lse, top[rows % D])
    dx, dw = pkg.linear_xent_bwd(x, w, target, lse, torch.ones(N, device=cuda))
    assert dx.float().abs().max().item() <= math.exp(-59) * V * w.float().abs().max().item()
    assert dw.float().abs().max().item() <= math.exp(-59) * N
    w[(t + 1) % V, cols] = w[t, cols]
    loss, lse = pkg.linear_xent(x, w, target, return_lse=True)
    _within(loss, math.log(2), 2.0 ** -24)
    want = top[rows % D].double() + math.log(2)
    _within(lse, want, 2.0 ** -24 * want.abs() + 2.0 ** -24)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logits_of_thousands(pkg, cuda, dtype):
    """Exact logits of standard deviation 400, against the formulas.  loss: rounded
    beside the maximum's distance from the target, 2 units of it.  lse is off by half a
    unit, 2^-24 of itself, which the probabilities take as a factor; the difference from
    a logit, its product and the exponential add 2^-24 of the exponent each (as far as p
    is not below 2^-150: at most 104 in size) and 2^-22."""
    N, V = 200, 900
    x, w, t = _exact(cuda, N, V, dtype, 4, 400.0)
    gen = torch.Generator(device=cuda).manual_seed(3)
    t = torch.randint(0, V, (N,), generator=gen, device=cuda)
    dloss = 0.5 + torch.rand(N, generator=gen, device=cuda)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    want, want_lse, wx, ww, sizes = oracle(x, w, t, dloss)
    _within(lse, want_lse, 2.0 ** -22 + 2.0 ** -24 * want_lse.abs())
    _within(loss, want, 2.0 ** -22 + 2.0 ** -23 * want)
    l = x.double() @ w.double().T
    p = torch.exp(l - want_lse[:, None])
    off = p * dloss.double()[:, None] * (2.0 ** -24 * want_lse.abs()[:, None] + 2 * 104 * 2.0 ** -24 + 2.0 ** -22)
    offs = ((off.square() @ w.double().square()).sum().sqrt().item(), (off.square().T @ x.double().square()).sum().sqrt().item())
    _close(dx, wx, 1.5, (sizes[0][0], offs[0]), "dx")
    _close(dw, ww, 1.5, (sizes[1][0], offs[1]), "dw")


# dloss, and the size of the operand that brings the gradient into fp16's range
SIZES = [(2.0 ** -30, 2.0 ** 13), (2.0 ** -16, 2.0 ** 8), (1.0, 1.0), (2.0 ** 16, 2.0 ** -8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("f,c", SIZES)
@pytest.mark.parametrize("which", ["dx", "dw"])
def test_dloss_of_every_size(pkg, cuda, dtype, f, c, which):
    """The unit of G follows dloss: a mean over many rows, a loss scale.  One operand is
    as large as makes its gradient a number of fp16, the other as small as keeps the
    logits."""
    gen = torch.Generator(device=cuda).manual_seed(6)
    N, V = 1100, 1100
    x, w = torch.randn(N, D, generator=gen, device=cuda), torch.randn(V, D, generator=gen, device=cuda)
    a, b = (0.25 / c, c) if which == "dx" else (c, 0.25 / c)
    x, w = (x * a).to(dtype), (w * b).to(dtype)
    t = torch.randint(0, V, (N,), generator=gen, device=cuda)
    dloss = f * (0.5 + torch.rand(N, generator=gen, device=cuda))
    lse = pkg.linear_xent(x, w, t, return_lse=True)[1]
    got = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    _, _, wx, ww, sizes = oracle(x, w, t, dloss)
    i = 0 if which == "dx" else 1
    want = (wx, ww)[i]
    assert want.norm() > 100 * 2.0 ** -25 * want.numel() ** 0.5       # (more than fp16's steps near zero)
    _close(got[i], want, 1.5, sizes[i], which)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_dloss_that_is_not_finite_stays_its_rows(pkg, cuda, dtype, bad):
    """The other rows' gradients as without it, though G has one unit for all."""
    x, w, t, dloss = _inputs(cuda, 200, 64, 1500, dtype, 4)
    w, x, dloss = (w.float() * 2 ** 12).to(dtype), (x.float() / 2 ** 12).to(dtype), dloss / 2 ** 10
    lse = pkg.linear_xent(x, w, t, return_lse=True)[1]
    keep = torch.arange(200, device=cuda) != 7
    wx, sizes = oracle(x, w, t, dloss)[2::2]
    dloss[7] = bad
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, dloss)
    _close(dx[keep], wx[keep], 1.5, sizes[0], "dx")
    assert not torch.isfinite(dx[7]).any() and not torch.isfinite(dw[t[7]]).any()


def test_a_million_rows_of_a_large_vocabulary(pkg, cuda):
    """More logits than the smallest tiles' launch would hold: forward and backward,
    some rows (the last among them) and some words against the formulas."""
    N, V, K = 1_000_000, 151_936, 8
    gen = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(N, K, generator=gen, device=cuda).bfloat16()
    w = torch.randn(V, K, generator=gen, device=cuda).bfloat16()
    t = torch.randint(-1000, V, (N,), generator=gen, device=cuda)
    loss, lse = pkg.linear_xent(x, w, t, return_lse=True)
    some = torch.cat([torch.randint(0, N, (100,), generator=gen, device=cuda), torch.arange(N - 100, N, device=cuda)])
    ones = torch.ones(1, device=cuda).expand(N)
    want, want_lse, wx, _, sizes = oracle(x[some], w, t[some], ones[some])
    _losses(loss[some], lse[some], want, want_lse)
    dx, dw = pkg.linear_xent_bwd(x, w, t, lse, ones)
    _close(dx[some], wx, 1.5, sizes[0], "dx")
    words = torch.cat([torch.arange(20, device=cuda), torch.arange(V - 20, V, device=cuda)])
    counts = (t >= 0)[:, None]
    g = torch.where(counts, torch.exp(x.double() @ w[words].double().T - lse.double()[:, None]), 0.0)
    off = g * 2.0 ** -15 * (1 + lse.abs())[:, None]
    g -= (t[:, None] == words).double()
    sq = lambda z: (z.square().T @ x.double().square()).sum().sqrt().item()
    _close(dw[words], g.T @ x.double(), 1.5, (sq(g), sq(off)), "dw")
