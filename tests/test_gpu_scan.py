"""GPU tests of gated_scan and gated_scan_bwd against the recurrence in 64 bits,
row by row.

Tolerances (2-norm of the difference over that of the result): the kernels
hold states and sums in fp32, so an fp32 output is within 2^-18 (64 roundings
of 2^-24: a state passes a few dozen products and sums that do not decay with
it) and a 16-bit one within that and one rounding to its type."""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -18
EPS = {torch.float16: 2.0 ** -11 + F32, torch.bfloat16: 2.0 ** -8 + F32, torch.float32: F32}


def _err(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.isfinite(got).all()
    n = want.norm()
    return ((got - want).norm() / n).item() if n > 0 else (got - want).norm().item()


def oracle(x, g, h0, dy, dfinal, lens):
    """64-bit recurrence and its gradient, sequence by sequence (lens: rows of
    the packed sequences, or None)."""
    x, g, dy = (t.double().cpu() for t in (x, g, dy))
    B, T, D = x.shape
    a = torch.exp(g)
    y, dx, dg = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    spans = [(b, 0, T) for b in range(B)] if lens is None else \
        [(0, s, s + n) for s, n in zip(itertools.accumulate([0] + lens[:-1]), lens)]
    N = len(spans)
    fs = torch.zeros(N, D, dtype=torch.float64) if h0 is None else h0.double().cpu().clone()
    dh0 = torch.zeros(N, D, dtype=torch.float64) if dfinal is None else dfinal.double().cpu().clone()
    for n, (b, s, e) in enumerate(spans):
        prev = []
        for t in range(s, e):
            prev.append(fs[n].clone())
            fs[n] = a[b, t] * fs[n] + x[b, t]
            y[b, t] = fs[n]
        for t in reversed(range(s, e)):
            dh = dy[b, t] + dh0[n]
            dx[b, t] = dh
            dg[b, t] = dh * a[b, t] * prev[t - s]
            dh0[n] = a[b, t] * dh
    return y, fs, dx, dg, dh0


def _inputs(dev, B, T, D, xd, gd, n, seed, gate=0.3, pad=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    wide = lambda t, dt: torch.cat([t, torch.full((B, T, pad), float("nan"))], -1).to(dt).to(dev)[..., :D] if pad else t.to(dt).to(dev)
    return (wide(rn(B, T, D), xd), wide(gate * torch.nn.functional.logsigmoid(rn(B, T, D)), gd),
            rn(n, D).to(dev), wide(rn(B, T, D), xd), rn(n, D).to(dev))


def _check(pkg, x, g, h0, dy, dfinal, lens, states):
    cu = None
    if lens is not None:
        cu = torch.tensor([0] + list(itertools.accumulate(lens)), device=x.device)
    y, fs, st = pkg.gated_scan(x, g, h0, cu_seqlens=cu, return_states=True)
    dx, dg, dh0 = pkg.gated_scan_bwd(x, g, h0, dy, dfinal, cu_seqlens=cu, states=st if states else None)
    torch.cuda.synchronize()
    want = oracle(x, g, h0, dy, dfinal, lens)
    for name, got, ref in zip(("y", "fs", "dx", "dg", "dh0"), (y, fs, dx, dg, dh0), want):
        assert got.shape == ref.shape
        if ref.numel():
            assert _err(got, ref) <= EPS[got.dtype], name


TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("xd,gd", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 1, 130), (3, 7, 64), (1, 8, 257), (2, 9, 128), (1, 128, 66),
                                   (2, 129, 33), (1, 500, 200), (2, 2049, 3), (1, 2500, 136)])
def test_dense(pkg, cuda, xd, gd, B, T, D):
    x, g, h0, dy, df = _inputs(cuda, B, T, D, xd, gd, B, seed=T + D)
    _check(pkg, x, g, h0, dy, df, None, states=True)


@pytest.mark.parametrize("T", [5, 100, 700])
def test_without_states(pkg, cuda, T):
    x, g, h0, dy, df = _inputs(cuda, 2, T, 70, torch.float32, torch.float32, 2, seed=1)
    _check(pkg, x, g, h0, dy, df, None, states=False)
    _check(pkg, x, g, None, dy, None, None, states=False)


@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [128, 128], [127, 129, 1, 0, 300], [3] * 90, [1000, 0, 1],
                                  [0, 0, 640]])
@pytest.mark.parametrize("D", [64, 77])
def test_packed(pkg, cuda, lens, D):
    x, g, h0, dy, df = _inputs(cuda, 1, sum(lens), D, torch.bfloat16, torch.float32, len(lens), seed=len(lens))
    _check(pkg, x, g, h0, dy, df, lens, states=True)
    _check(pkg, x, g, h0, dy, df, lens, states=False)


@pytest.mark.parametrize("T", [1, 8, 9, 300])
def test_strides(pkg, cuda, T):
    """Rows inside wider rows of NaN, odd and even pads; batches out of order."""
    for pad in (1, 2, 7):
        x, g, h0, dy, df = _inputs(cuda, 3, T, 66, torch.float16, torch.float16, 3, seed=pad, pad=pad)
        x, g, dy = (t.flip(0).transpose(0, 1).contiguous().transpose(0, 1) if pad == 7 else t for t in (x, g, dy))
        _check(pkg, x, g, h0, dy, df, None, states=True)


def test_misaligned_pointer(pkg, cuda):
    x, g, h0, dy, df = _inputs(cuda, 1, 200, 64, torch.bfloat16, torch.bfloat16, 1, seed=9)
    off = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view_as(t)
    _check(pkg, off(x), off(g), h0, off(dy), df, None, states=True)


@pytest.mark.parametrize("T", [6, 400])
def test_gates_at_their_ends(pkg, cuda, T):
    """g = -inf forgets the state (later rows do not see earlier ones), g = 0
    keeps it; a NaN or an infinity in one sequence or channel stays there."""
    x, g, h0, dy, df = _inputs(cuda, 2, T, 64, torch.float32, torch.float32, 2, seed=3)
    g[:, T // 2] = float("-inf")
    g[:, T // 3] = 0.0
    _check(pkg, x, g, h0, dy, df, None, states=True)
    clean, _ = pkg.gated_scan(x, g, h0)
    x2, h2 = x.clone(), h0.clone()
    x2[0, 1, 5] = float("nan")
    h2[0, 7] = float("inf")
    y, fs = pkg.gated_scan(x2, g, h2)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[0, 1:, 5] = True
    hit[0, :, 7] = True
    assert torch.equal(y[~hit], clean[~hit])
    assert torch.isinf(y[0, : T // 3, 7]).all() and torch.isnan(y[0, 1:, 5]).all()


def test_strong_and_weak_gates(pkg, cuda):
    """Gates of the benchmark's recipe, and gates so near 1 that a state lives
    through every row."""
    for gate in (1.0, 8.0, 1e-4):
        x, g, h0, dy, df = _inputs(cuda, 1, 1500, 40, torch.float32, torch.float32, 1, seed=4, gate=gate)
        _check(pkg, x, g, h0, dy, df, None, states=True)


def test_offsets_past_32_bits(pkg, cuda):
    """Rows whose element offset passes 2^31: batch stride beyond 2^30."""
    D, T = 16, 40
    big = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.float16, device=cuda)
    x = torch.as_strided(big, (2, T, D), (2 ** 31 - 4096, D * 3, 1))
    gen = torch.Generator(device=cuda).manual_seed(1)
    x.copy_(torch.randn(2, T, D, generator=gen, device=cuda))
    g = -torch.rand(2, T, D, generator=gen, device=cuda)
    h0 = torch.randn(2, D, generator=gen, device=cuda)
    y, fs = pkg.gated_scan(x, g, h0)
    y2, fs2 = pkg.gated_scan(x.contiguous(), g, h0)
    assert torch.equal(y, y2) and torch.equal(fs, fs2)


def test_autograd_and_differences(pkg, cuda):
    """Autograd's gradients equal gated_scan_bwd's, and agree with central
    differences of a scalar of both outputs."""
    x, g, h0, dy, df = _inputs(cuda, 2, 150, 32, torch.float32, torch.float32, 2, seed=8)
    xs, gs, hs = (t.clone().requires_grad_() for t in (x, g, h0))
    y, fs = pkg.gated_scan(xs, gs, hs)
    ((y * dy).sum() + (fs * df).sum()).backward()
    dx, dg, dh0 = pkg.gated_scan_bwd(x, g, h0, dy, df)
    for a, b in ((xs.grad, dx), (gs.grad, dg), (hs.grad, dh0)):
        assert _err(a, b) <= F32
    f = lambda x, g, h0: ((lambda r: (r[0].double() * dy).sum() + (r[1].double() * df).sum())(pkg.gated_scan(x, g, h0))).item()
    gen = torch.Generator(device=cuda).manual_seed(2)
    for i, (t, grad) in enumerate(((x, dx), (g, dg), (h0, dh0))):
        v = torch.randn(t.shape, generator=gen, device=cuda)
        eps = 2.0 ** -7
        args = [x, g, h0]
        up, down = (f(*(args[:i] + [t + s * eps * v] + args[i + 1:])) for s in (1, -1))
        want = (grad.double() * v).sum().item()
        # third-order terms of e^g (eps^2) and fp32 roundings over eps
        assert abs((up - down) / (2 * eps) - want) <= 2.0 ** -9 * (grad.norm() * v.norm()).item()


def test_only_some_gradients(pkg, cuda):
    x, g, h0, dy, df = _inputs(cuda, 1, 64, 8, torch.float32, torch.float32, 1, seed=8)
    x.requires_grad_()
    y, fs = pkg.gated_scan(x, g)
    fs.sum().backward()
    want = oracle(x.detach(), g, None, torch.zeros_like(g), torch.ones(1, 8), None)[2]
    assert _err(x.grad, want) <= F32


def test_other_stream_and_graph(pkg, cuda):
    """The call runs on the current stream and can be captured; replays give
    the eager result for new inputs in the same buffers."""
    x, g, h0, _, _ = _inputs(cuda, 2, 300, 64, torch.bfloat16, torch.float32, 2, seed=5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y1, _ = pkg.gated_scan(x, g, h0)
    torch.cuda.current_stream().wait_stream(s)
    y0, _ = pkg.gated_scan(x, g, h0)
    assert torch.equal(y0, y1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg, fg = pkg.gated_scan(x, g, h0)
    for k in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        y, fs = pkg.gated_scan(x, g, h0)
        assert torch.equal(y, yg) and torch.equal(fs, fg)


def test_repeatable(pkg, cuda):
    x, g, h0, dy, df = _inputs(cuda, 1, 5000, 256, torch.bfloat16, torch.float32, 1, seed=5)
    runs = [(*pkg.gated_scan(x, g, h0), *pkg.gated_scan_bwd(x, g, h0, dy, df)) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.parametrize("gate", [0.3, 2.0, 8.0])
@pytest.mark.parametrize("xd,gd", TYPES)
def test_infinite_states_stay(pkg, cuda, xd, gd, gate):
    """An infinite state stays infinite under finite gates however many rows it
    lives through, forward and backward, and a gate of -inf makes it NaN as
    0 inf is; other channels keep their bits."""
    T = 2500
    x, g, h0, dy, df = _inputs(cuda, 2, T, 66, xd, gd, 2, seed=51, gate=gate)
    y, fs, st = pkg.gated_scan(x, g, h0, return_states=True)
    dx, dg, dh0 = pkg.gated_scan_bwd(x, g, h0, dy, df, states=st)
    x2, h2, df2, dy2 = x.clone(), h0.clone(), df.clone(), dy.clone()
    inf = float("inf")
    h2[0, 7], h2[1, 8], x2[0, 300, 9] = inf, -inf, inf
    df2[0, 20], dy2[1, 2000, 21] = -inf, inf
    y2, fs2, st2 = pkg.gated_scan(x2, g, h2, return_states=True)
    assert (y2[0, :, 7] == inf).all() and (y2[1, :, 8] == -inf).all() and (y2[0, 300:, 9] == inf).all()
    assert fs2[0, 7] == inf and fs2[1, 8] == -inf and fs2[0, 9] == inf
    hit = torch.zeros_like(y2, dtype=torch.bool)
    hit[0, :, 7] = hit[1, :, 8] = hit[0, 300:, 9] = True
    assert torch.equal(y2[~hit], y[~hit])
    for states in (st, None):
        dx2, _, dh2 = pkg.gated_scan_bwd(x, g, h0, dy2, df2, states=states)
        assert (dx2[0, :, 20] == -inf).all() and (dx2[1, :2001, 21] == inf).all()
        assert dh2[0, 20] == -inf and dh2[1, 21] == inf
        hit = torch.zeros_like(dx2, dtype=torch.bool)
        hit[0, :, 20] = hit[1, :2001, 21] = True
        assert torch.equal(dx2[~hit], dx[~hit])
    g2 = g.clone()
    g2[0, 900, 7] = -inf
    y2, _ = pkg.gated_scan(x2, g2, h2)
    assert (y2[0, :900, 7] == inf).all() and torch.isnan(y2[0, 900:, 7]).all()


def test_growing_gates_before_any_state(pkg, cuda):
    """Gates above 0 over rows whose state is still zero: e^G of many rows leaves
    the range of floats, the rows' own states do not."""
    x, g, _, dy, _ = _inputs(cuda, 1, 2600, 64, torch.float32, torch.float32, 1, seed=52)
    g[:, :2200] = 0.5
    x[:, :2200] = 0.0
    y, fs = pkg.gated_scan(x, g)
    want = oracle(x, g, None, dy, None, None)
    assert _err(y, want[0]) <= F32 and _err(fs, want[1]) <= F32


def test_states_of_another_call_are_refused(pkg, cuda):
    x, g, h0, dy, df = _inputs(cuda, 1, 300, 64, torch.float32, torch.float32, 1, seed=9)
    _, _, st = pkg.gated_scan(x, g, h0, return_states=True)
    for bad in ("states", 3, st[:-1], st.double(), st.t().contiguous().t(), st.cpu()):
        with pytest.raises(ValueError):
            pkg.gated_scan_bwd(x, g, h0, dy, df, states=bad)
