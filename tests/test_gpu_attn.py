"""GPU tests of window_attn, window_attn_bwd and window_attn_decode against the
formulas in 64 bits, row by row of the mask.

Tolerances (2-norm of the difference over that of the result): an output is
rounded once to its type, and the probabilities and dS are rounded once to the
operand type before the sums that they enter (fp32 elsewhere); the roundings
are independent, so an output with one operand rounding is within 1.5 of its
type's unit.  dS = P (dP - D) takes D from the rounded o and cancels where one
key dominates: gradients get 4 units of the size of the terms that enter them,
here that of the result or, for rows with few keys, of sum |P dP|."""

import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]


def visible(T, S, window, sinks, dev):
    p = (S - T + torch.arange(T, device=dev))[:, None]
    j = torch.arange(S, device=dev)[None]
    m = j <= p
    if window is not None:
        m &= (j > p - window) | (j < sinks)
    return m


def oracle(q, k, v, window, sinks, scale=None, do=None):
    """One sequence, [T, Hq, D] and [S, Hk, D]; masked places take part in
    nothing, whatever they hold."""
    T, Hq, D = q.shape
    S, Hk = k.shape[:2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.double() for t in (q, k, v))
    m = visible(T, S, window, sinks, q.device)
    o = torch.zeros_like(q)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    grads = None
    if do is not None:
        do = do.double()
        grads = [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
        sizes = [torch.zeros_like(q), torch.zeros_like(k)]
    for h in range(Hq):
        K, V = k[:, h // G], v[:, h // G]
        s = torch.where(m, q[:, h] @ K.T * scale, -math.inf)
        lse[:, h] = torch.logsumexp(s, -1)
        top = s.amax(-1, keepdim=True) if S else s.new_full((T, 1), -math.inf)
        p = torch.where(m, torch.exp(s - torch.where(top > -math.inf, top, 0.0)), 0.0)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        o[:, h] = p @ V
        if do is not None:
            dp = do[:, h] @ V.T
            delta = (do[:, h] * o[:, h]).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            grads[0][:, h] = ds @ K
            grads[1][:, h // G] += ds.T @ q[:, h]
            grads[2][:, h // G] += p.T @ do[:, h]
            t = p * (dp.abs() + delta.abs()) * scale
            sizes[0][:, h] = t.square() @ K.square()
            sizes[1][:, h // G] += t.square().T @ q[:, h].square()
    if do is None:
        return o, lse
    return o, lse, grads, [x.sum().sqrt().item() for x in sizes]


def _close(got, want, units, size=0.0, name=""):
    assert torch.isfinite(got).all(), name
    d = (got.double() - want).norm().item()
    n = max(want.norm().item(), size)
    assert d <= units * UNIT[got.dtype] * n + 1e-30, (name, d / max(n, 1e-30) / UNIT[got.dtype])


def _inputs(dev, B, T, S, Hq, Hk, D, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev)
    return (rn(B, T, Hq, D).to(dtype), rn(B, S, Hk, D).to(dtype), rn(B, S, Hk, D).to(dtype), rn(B, T, Hq, D).to(dtype))


def _check(pkg, q, k, v, do, window, sinks, scale=None, lens=None, backward=True):
    cu = None
    if lens is not None:
        cu = torch.tensor([0] + list(itertools.accumulate(lens)), device=q.device)
    o, lse = pkg.window_attn(q, k, v, window, sinks, scale, cu_seqlens=cu, return_lse=True)
    if backward:
        dq, dk, dv = pkg.window_attn_bwd(q, k, v, o, lse, do, window, sinks, scale, cu_seqlens=cu)
    torch.cuda.synchronize()
    at = [(b, 0, q.shape[1]) for b in range(q.shape[0])] if lens is None else \
        [(0, s, s + n) for s, n in zip(itertools.accumulate([0] + lens[:-1]), lens)]
    for b, s, e in at:
        if lens is not None and s == e:
            continue
        ks = slice(s, e) if lens is not None else slice(None)
        args = (q[b, s:e], k[b, ks], v[b, ks], window, sinks, scale)
        if not backward:
            wo, wl = oracle(*args)
        else:
            wo, wl, (wq, wk, wv), (sq, sk) = oracle(*args, do=do[b, s:e])
        _close(o[b, s:e], wo, 1.5, name="o")
        got = lse[b, s:e].double()
        none = wl == -math.inf
        assert torch.equal(got == -math.inf, none)
        # scores are sums of D products in fp32
        assert ((got - wl)[~none].abs() <= 2.0 ** -15 * (1 + wl[~none].abs())).all()
        assert (o[b, s:e][none] == 0).all()
        if backward:
            _close(dq[b, s:e], wq, 4, sq, "dq")
            _close(dk[b, ks], wk, 4, sk, "dk")
            _close(dv[b, ks], wv, 2, 0.0, "dv")
            assert (dq[b, s:e][none] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,window,sinks", [(1, None, 0), (2, 1, 0), (31, 7, 1), (64, 64, 0), (65, 16, 4), (128, None, 0),
                                            (129, 128, 0), (200, 33, 3), (300, 64, 70), (515, 100, 4), (700, 1, 0),
                                            (777, 50, 200), (1030, 300, 5)])
def test_dense(pkg, cuda, dtype, D, T, window, sinks):
    q, k, v, do = _inputs(cuda, 2, T, T, 4, 2, D, dtype, seed=T)
    _check(pkg, q, k, v, do, window, sinks)


@pytest.mark.parametrize("B,Hq,Hk", [(1, 1, 1), (3, 3, 1), (1, 8, 8), (2, 12, 4), (1, 10, 2), (4, 4, 2)])
def test_heads(pkg, cuda, B, Hq, Hk):
    q, k, v, do = _inputs(cuda, B, 333, 333, Hq, Hk, 64, torch.bfloat16, seed=Hq)
    _check(pkg, q, k, v, do, 90, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,S", [(1, 500), (3, 64), (100, 400), (130, 129), (200, 70), (300, 1), (5, 0), (0, 40), (64, 1000)])
def test_more_or_fewer_keys(pkg, cuda, dtype, T, S):
    """Query rows at the end of longer keys; more rows than keys, where the
    first see none; no rows and no keys."""
    q, k, v, do = _inputs(cuda, 2, T, S, 4, 2, 64, dtype, seed=T + S)
    for window, sinks in ((None, 0), (50, 3)):
        _check(pkg, q, k, v, do, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[1], [0, 7, 0], [128, 128], [127, 1, 0, 300, 129], [5] * 40, [900, 64, 1]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 0), (40, 5), (3, 150)])
def test_packed(pkg, cuda, dtype, lens, window, sinks):
    T = sum(lens)
    q, k, v, do = _inputs(cuda, 1, T, T, 4, 2, 64, dtype, seed=T)
    _check(pkg, q, k, v, do, window, sinks, lens=lens)


@pytest.mark.parametrize("sinks", [1, 130, 600])
def test_many_segments_of_the_first_keys(pkg, cuda, sinks):
    q, k, v, do = _inputs(cuda, 1, 3000, 3000, 2, 1, 128, torch.bfloat16, seed=sinks)
    _check(pkg, q, k, v, do, 16, sinks)
    q, k, v, do = _inputs(cuda, 1, 3000, 3000, 2, 1, 64, torch.float16, seed=sinks)
    _check(pkg, q, k, v, do, 16, sinks, lens=[1400, 3, 1597])


def test_strides_and_scale(pkg, cuda):
    """[B, H, T, D] memory, heads inside wider rows, one projection cut in three."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda).to(torch.bfloat16)
    q, k, v, do = (rn(2, h, 200, 64).transpose(1, 2) for h in (4, 2, 2, 4))
    _check(pkg, q, k, v, do, 77, 2, scale=0.3)
    qkv = rn(2, 200, 8, 72)[..., :64]
    _check(pkg, qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:], do, 77, 2, scale=-0.2)
    _check(pkg, rn(1, 200, 4, 64).expand(2, -1, -1, -1), k, v, do, None, 0)


def test_offsets_past_32_bits(pkg, cuda):
    big = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.float16, device=cuda)
    k = torch.as_strided(big, (2, 100, 1, 64), (2 ** 31 - 2 ** 14, 128, 64, 1))
    gen = torch.Generator(device=cuda).manual_seed(1)
    k.copy_(torch.randn(2, 100, 1, 64, generator=gen, device=cuda))
    q, _, v, do = _inputs(cuda, 2, 100, 100, 2, 1, 64, torch.float16, seed=2)
    _check(pkg, q, k, v, do, 30, 1)
    # rows so far apart that a tile spans more than 2^31 bytes
    k = torch.as_strided(big, (1, 100, 1, 64), (0, 2 ** 24 + 8, 64, 1))
    k.copy_(torch.randn(1, 100, 1, 64, generator=gen, device=cuda))
    _check(pkg, q[:1], k, v[:1], do[:1], 30, 1)
    o = pkg.window_attn_decode(q[:1, :2], k, v[:1], torch.tensor([97], device=cuda, dtype=torch.int32), 30, 1)
    _close(o[0], oracle(q[0, :2], k[0, :97], v[0, :97], 30, 1)[0], 1.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_not_finite_places_stay_hidden(pkg, cuda, dtype, D, value):
    """A key, value, query or gradient row that is not finite reaches the rows
    that see it and no others."""
    T, window, sinks = 300, 40, 3
    q, k, v, do = _inputs(cuda, 1, T, T, 2, 1, D, dtype, seed=3)
    clean = pkg.window_attn(q, k, v, window, sinks, return_lse=True)
    gclean = pkg.window_attn_bwd(q, k, v, *clean, do, window, sinks)
    m = visible(T, T, window, sinks, cuda)
    for j in (0, 130, 199, 299):
        hit = m[:, j]
        for which in ("k", "v"):
            k2, v2 = k.clone(), v.clone()
            (k2 if which == "k" else v2)[0, j, 0, 5] = value
            o, lse = pkg.window_attn(q, k2, v2, window, sinks, return_lse=True)
            assert torch.equal(o[0, ~hit], clean[0][0, ~hit]), (which, j)
            if which == "v":
                want = torch.full_like(o[0, hit, :, 5], value)
                assert torch.equal(o[0, hit, :, 5].isnan(), want.isnan())
                if not math.isnan(value):
                    assert torch.equal(o[0, hit, :, 5], want)
                assert torch.isfinite(o[0][..., :5]).all()
            elif math.isnan(value):
                assert torch.isnan(o[0, hit]).all()
            dq, dk, dv = pkg.window_attn_bwd(q, k2, v2, o, lse, do, window, sinks)
            assert torch.equal(dq[0, ~hit], gclean[0][0, ~hit]), (which, j)
            far = ~m[hit].any(0)          # keys that no hit row sees
            assert torch.equal(dk[0, far], gclean[1][0, far]) and torch.equal(dv[0, far], gclean[2][0, far])
    for i in (0, 131, 299):
        seen = m[i]
        q2 = q.clone()
        q2[0, i, 0, 7] = value
        o, lse = pkg.window_attn(q2, k, v, window, sinks, return_lse=True)
        rest = torch.arange(T, device=cuda) != i
        assert torch.equal(o[0, rest], clean[0][0, rest])
        dq, dk, dv = pkg.window_attn_bwd(q2, k, v, o, lse, do, window, sinks)
        assert torch.equal(dq[0, rest], gclean[0][0, rest])
        assert torch.equal(dk[0, ~seen], gclean[1][0, ~seen]) and torch.equal(dv[0, ~seen], gclean[2][0, ~seen])
        do2 = do.clone()
        do2[0, i, 1, 9] = value
        dq, dk, dv = pkg.window_attn_bwd(q, k, v, *clean, do2, window, sinks)
        assert torch.equal(dq[0, rest], gclean[0][0, rest])
        assert torch.equal(dk[0, ~seen], gclean[1][0, ~seen]) and torch.equal(dv[0, ~seen], gclean[2][0, ~seen])
        assert not torch.isfinite(dv[0, seen, 0, 9]).any()


@pytest.mark.parametrize("p", [4, 10, 14])
def test_small_gradients(pkg, cuda, p):
    """dO of rows far below the rest, and all of it: fp16 keeps the gradients'
    precision by their own size (the rounded results are subnormal at 2^-14
    and are compared with that step)."""
    T = 400
    for dtype in DTYPES:
        q, k, v, do = _inputs(cuda, 1, T, T, 2, 1, 64, dtype, seed=p)
        q, k = q * 8, k
        do = do * 2.0 ** -p
        o, lse = pkg.window_attn(q, k, v, 100, 0, return_lse=True)
        got = pkg.window_attn_bwd(q, k, v, o, lse, do, 100, 0)
        _, _, want, sizes = oracle(q[0], k[0], v[0], 100, 0, do=do[0])
        floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
        for g, w, s, name in zip(got, want, (*sizes, 0.0), ("dq", "dk", "dv")):
            d = (g[0].double() - w).norm().item()
            assert d <= 4 * UNIT[dtype] * max(w.norm().item(), s) + floor * math.sqrt(w.numel()), name
        # one half of the rows much smaller: its dq by its own size
        do2 = do * 2.0 ** p
        do2[:, :200] *= 2.0 ** -8
        got = pkg.window_attn_bwd(q, k, v, o, lse, do2, 100, 0)
        _, _, want, _ = oracle(q[0], k[0], v[0], 100, 0, do=do2[0])
        d = (got[0][0, :200].double() - want[0][:200]).norm().item()
        assert d <= 6 * UNIT[dtype] * want[0][:200].norm().item() + floor * math.sqrt(want[0][:200].numel())


def test_large_values_fp16(pkg, cuda):
    """fp16 v and dO near the type's end: no overflow on the way."""
    q, k, v, do = _inputs(cuda, 1, 200, 200, 2, 1, 64, torch.float16, seed=6)
    v, do = v * 300, do * 30
    o, lse = pkg.window_attn(q * 0.1, k, v, 50, 0, return_lse=True)
    dq, dk, dv = pkg.window_attn_bwd(q * 0.1, k, v, o, lse, do, 50, 0)
    _, _, want, sizes = oracle((q * 0.1)[0], k[0], v[0], 50, 0, do=do[0])
    for g, w, s, name in zip((dq, dk, dv), want, (*sizes, 0.0), ("dq", "dk", "dv")):
        fits = w.abs() < 60000
        assert torch.isfinite(g[0][fits]).all()
        d = ((g[0].double() - w)[fits]).norm().item()
        assert d <= 4 * UNIT[torch.float16] * max(w[fits].norm().item(), s), name


def test_large_scores(pkg, cuda):
    """Scores whose exponentials leave fp32, falling and rising along the keys."""
    q, k, v, do = _inputs(cuda, 1, 300, 300, 2, 1, 64, torch.bfloat16, seed=5)
    ramp = torch.linspace(0.1, 40, 300, device=cuda)
    for r in (ramp, ramp.flip(0)):
        k2 = (k * r[None, :, None, None]).to(k.dtype)
        _check(pkg, q * 4, k2, v, do, None, 0, backward=False)
        _check(pkg, q * 4, k2, v, do, 70, 2, backward=False)


def _decode_check(pkg, q, kc, vc, lens, window, sinks):
    o = pkg.window_attn_decode(q, kc, vc, torch.tensor(lens, dtype=torch.int32, device=q.device), window, sinks)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        wo, _ = oracle(q[b], kc[b, :n], vc[b, :n], window, sinks)
        _close(o[b], wo, 1.5, name=f"sequence {b} of {n}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hq,Hk", [(1, 4, 4), (1, 16, 4), (2, 6, 2), (1, 40, 1), (16, 12, 3), (5, 1, 1)])
def test_decode(pkg, cuda, dtype, D, T, Hq, Hk):
    lens = [T, 33, 64, 500, 1000, 31, 32, 999]
    q, kc, vc, _ = _inputs(cuda, len(lens), T, 1000, Hq, Hk, D, dtype, seed=T + Hq)
    for b, n in enumerate(lens):        # what lies past the keys is never read
        kc[b, n:] = float("nan")
        vc[b, n:] = float("inf")
    for window, sinks in ((None, 0), (100, 4), (1, 0), (64, 200)):
        _decode_check(pkg, q, kc, vc, lens, window, sinks)


def test_decode_short_and_empty(pkg, cuda):
    """No keys at all, fewer keys than tokens, lengths outside the cache."""
    q, kc, vc, _ = _inputs(cuda, 4, 4, 50, 4, 2, 64, torch.bfloat16, seed=1)
    lens = torch.tensor([0, 2, -5, 80], dtype=torch.int64, device=cuda)
    o = pkg.window_attn_decode(q, kc, vc, lens, 20, 1)
    assert (o[0] == 0).all() and (o[2] == 0).all() and (o[1, :2] == 0).all()
    for b, n in ((1, 2), (3, 50)):
        _close(o[b], oracle(q[b], kc[b, :n], vc[b, :n], 20, 1)[0], 1.5)


def test_decode_long_cache(pkg, cuda):
    """A cache of more than 2^31 elements, one sequence deep inside it."""
    S = 2 ** 17
    kc = torch.zeros(1, S, 136, 128, dtype=torch.bfloat16, device=cuda)[:, :, 128:136]
    gen = torch.Generator(device=cuda).manual_seed(1)
    kc[:, -6000:] = torch.randn(1, 6000, 8, 128, generator=gen, device=cuda).to(torch.bfloat16)
    q = torch.randn(1, 1, 16, 128, generator=gen, device=cuda).to(torch.bfloat16)
    n = S - 7
    o = pkg.window_attn_decode(q, kc, kc, torch.tensor([n], device=cuda), 5000, 2)
    keys = torch.cat([kc[0, :2], kc[0, n - 5000:n]])
    want, _ = oracle(q[0], keys, keys, None, 0)
    _close(o[0], want, 1.5)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_decode_hidden_rows(pkg, cuda, value):
    """Cache rows before the window may hold anything."""
    q, kc, vc, _ = _inputs(cuda, 2, 2, 400, 4, 2, 128, torch.float16, seed=1)
    lens = [400, 333]
    want = pkg.window_attn_decode(q, kc, vc, torch.tensor(lens, device=cuda), 50, 3)
    for b, n in enumerate(lens):
        kc[b, 3:n - 51] = value
        vc[b, 3:n - 51] = value
    got = pkg.window_attn_decode(q, kc, vc, torch.tensor(lens, device=cuda), 50, 3)
    assert torch.equal(got, want)
    # a row that only the older of two tokens sees
    vc[0, 400 - 51] = value
    got = pkg.window_attn_decode(q, kc, vc, torch.tensor(lens, device=cuda), 50, 3)
    assert torch.equal(got[0, 1], want[0, 1]) and not torch.isfinite(got[0, 0]).any()


def test_decode_equals_prefill(pkg, cuda):
    q, k, v, _ = _inputs(cuda, 2, 260, 260, 8, 2, 128, torch.bfloat16, seed=11)
    o = pkg.window_attn(q, k, v, 64, 4)
    for n in (1, 5, 68, 69, 260):
        got = pkg.window_attn_decode(q[:, n - 1:n], k, v, torch.tensor([n, n], device=cuda), 64, 4)
        _close(got, o[:, n - 1:n].double(), 2.0)


def test_autograd(pkg, cuda):
    q, k, v, do = _inputs(cuda, 2, 150, 150, 4, 2, 64, torch.bfloat16, seed=12)
    a, b, c = (t.clone().requires_grad_() for t in (q, k, v))
    o, lse = pkg.window_attn(a, b, c, 40, 2, return_lse=True)
    assert not lse.requires_grad
    o.backward(do)
    want = pkg.window_attn_bwd(q, k, v, o.detach(), lse, do, 40, 2)
    assert all(torch.equal(x.grad, y) for x, y in zip((a, b, c), want))
    # the expansion of a scalar as dO; gradients of one input only
    a.grad = None
    pkg.window_attn(a, k, v, 40, 2).float().sum().backward()
    want = pkg.window_attn_bwd(q, k, v, o.detach(), lse, torch.ones_like(do), 40, 2)
    assert torch.equal(a.grad, want[0])


def test_gradient_and_differences(pkg, cuda):
    """Directional derivative of the 64-bit oracle's output along random
    directions against the kernel's gradients."""
    q, k, v, do = _inputs(cuda, 1, 90, 90, 2, 1, 64, torch.float16, seed=13)
    o, lse = pkg.window_attn(q, k, v, 30, 2, return_lse=True)
    grads = pkg.window_attn_bwd(q, k, v, o, lse, do, 30, 2)
    gen = torch.Generator(device=cuda).manual_seed(3)
    f = lambda a, b, c: (oracle(a, b, c, 30, 2)[0] * do[0].double()).sum().item()
    args = [t[0].double() for t in (q, k, v)]
    for i, g in enumerate(grads):
        u = torch.randn(args[i].shape, generator=gen, device=cuda, dtype=torch.float64)
        step = 1e-5
        up, down = (f(*(args[:i] + [args[i] + s * step * u] + args[i + 1:])) for s in (1, -1))
        want = (up - down) / (2 * step)
        got = (g[0].double() * u).sum().item()
        assert abs(got - want) <= 4 * UNIT[torch.float16] * (g.double().norm() * u.norm()).item()


def test_stream_graph_and_repeat(pkg, cuda):
    q, k, v, do = _inputs(cuda, 1, 900, 900, 4, 2, 128, torch.bfloat16, seed=14)
    first = pkg.window_attn(q, k, v, 100, 4, return_lse=True)
    g1 = pkg.window_attn_bwd(q, k, v, *first, do, 100, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = pkg.window_attn(q, k, v, 100, 4, return_lse=True)
        g2 = pkg.window_attn_bwd(q, k, v, *again, do, 100, 4)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip((*first, *g1), (*again, *g2)))
    lens = torch.tensor([777], dtype=torch.int32, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        og = pkg.window_attn_decode(q[:, :1], k, v, lens, 200, 4)
        ag = pkg.window_attn(q, k, v, 100, 4)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        lens.fill_(400 + 100 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(og, pkg.window_attn_decode(q[:, :1], k, v, lens, 200, 4))
        assert torch.equal(ag, pkg.window_attn(q, k, v, 100, 4))


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_many_key_blocks(pkg, cuda, D, dtype):
    """Enough key blocks for workgroups of 4 waves (the smaller tests have the
    blocks shared by several)."""
    q, k, v, do = _inputs(cuda, 8, 700, 700, 12, 12, D, dtype, seed=21)
    _check(pkg, q, k, v, do, 130, 3)
    q, k, v, do = _inputs(cuda, 1, 5000, 5000, 16, 16, D, dtype, seed=22)
    _check(pkg, q, k, v, do, 200, 20, lens=[1999, 0, 1, 3000])


@pytest.mark.parametrize("D", [64, 128])
def test_gradient_over_few_keys(pkg, cuda, D):
    """Rows of few keys: D = sum P dP beside dP, where the rounding of o would
    show.  In packed sequences of 1 to 40 rows what is left is the rounding of dS
    and of the result, each uniform up to 2^-8: 3^-0.5 2^-8 each, (2 / 3)^0.5
    2^-8 of the norm together.  A row with one key has dq = 0 but for the sums'
    own rounding, 2^-20 of |dO| |v| |k|."""
    lens = [1, 3, 40, 1, 17, 8, 25, 2, 9]
    T, Hq, Hk = sum(lens), 4, 2
    gen = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(1, T, h, D, generator=gen).to(torch.bfloat16) for h in (Hq, Hk, Hk, Hq))
    cu = torch.tensor([0] + lens).cumsum(0)
    qc, kc, vc, dc = (t.to(cuda) for t in (q, k, v, do))
    o, lse = pkg.window_attn(qc, kc, vc, 16, 1, cu_seqlens=cu.to(cuda), return_lse=True)
    got = pkg.window_attn_bwd(qc, kc, vc, o, lse, dc, 16, 1, cu_seqlens=cu.to(cuda))
    want = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
    for s, e in zip(cu[:-1].tolist(), cu[1:].tolist()):
        x, kk, vv, dd = (t[0, s:e].double() for t in (q, k, v, do))
        kr, vr = kk.repeat_interleave(Hq // Hk, 1), vv.repeat_interleave(Hq // Hk, 1)
        sc = torch.einsum("thd,shd->hts", x, kr) * D ** -0.5
        i, j = torch.arange(e - s)[:, None], torch.arange(e - s)[None]
        P = sc.masked_fill(~((j <= i) & ((j > i - 16) | (j < 1))), -torch.inf).softmax(-1)
        dP = torch.einsum("thd,shd->hts", dd, vr)
        dS = P * (dP - (P * dP).sum(-1, keepdim=True)) * D ** -0.5
        want[0][0, s:e] = torch.einsum("hts,shd->thd", dS, kr)
        want[1][0, s:e] = torch.einsum("hts,thd->shd", dS, x).view(e - s, Hk, -1, D).sum(2)
        want[2][0, s:e] = torch.einsum("hts,thd->shd", P, dd).view(e - s, Hk, -1, D).sum(2)
    for g, w in zip(got, want):
        assert (g.cpu().double() - w).norm() <= (2 / 3) ** 0.5 * 2.0 ** -8 * w.norm()
    first = [s for s in cu[:-1].tolist()]
    size = (do[0, first].double().norm(dim=-1) * v[0, first].double().norm(dim=-1).repeat_interleave(2, -1)
            * k[0, first].double().norm(dim=-1).repeat_interleave(2, -1))
    assert (got[0][0, first].cpu().double().norm(dim=-1) <= 2.0 ** -20 * size).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,S,Hq,Hk,window,sinks", [(1, 20, 4001, 4, 2, None, 0), (2, 1, 3000, 2, 1, 1500, 3),
                                                      (1, 700, 1500, 2, 2, 400, 130), (1, 1100, 1100, 3, 1, None, 5),
                                                      (1, 900, 640, 2, 1, None, 0)])
def test_few_rows_over_long_keys(pkg, cuda, dtype, D, B, T, S, Hq, Hk, window, sinks):
    """Blocks whose keys are shared by several workgroups: splits that see no
    key, rows that see none at all, and infinities in hidden places of one split."""
    gen = torch.Generator().manual_seed(T + S)
    q, k, v = (torch.randn(B, n, h, D, generator=gen).to(dtype).to(cuda) for n, h in ((T, Hq), (S, Hk), (S, Hk)))
    seen = visible(T, S, window, sinks, cuda)
    hidden = ~seen.any(0)
    kk, vv = (t.repeat_interleave(Hq // Hk, 2).transpose(1, 2).double() for t in (k, v))
    s = torch.matmul(q.transpose(1, 2).double(), kk.transpose(2, 3).contiguous()) * D ** -0.5
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1).transpose(1, 2)
    P = torch.where(seen, torch.exp(s - torch.where(lse > -math.inf, lse, 0.0).transpose(1, 2)[..., None]), 0.0)
    want = torch.matmul(P, vv.contiguous()).transpose(1, 2)
    for value in (None, math.inf):
        if value is not None:
            if not hidden.any():
                continue
            v = v.clone()
            v[:, hidden] = value
        o, l = pkg.window_attn(q, k, v, window, sinks, return_lse=True)
        torch.cuda.synchronize()
        assert (o.double() - want).norm() <= 1.5 * UNIT[dtype] * want.norm()
        none = ~seen.any(1)
        assert (o[:, none] == 0).all() and (l[:, none] == -math.inf).all()
        assert (l[:, ~none].double() - lse[:, ~none]).abs().max() <= 2.0 ** -18 * max(1.0, lse[:, ~none].abs().max().item())


@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("T,lens", [(None, None), (7, None), (None, [0, 1, 0]), (None, [0, 0, 300])])
@pytest.mark.parametrize("window,sinks", [(128, 1), (128, 4), (60, 130), (1024, 4)])
@pytest.mark.parametrize("beyond", [127, 128, 129])
def test_first_rows_beyond_a_blocks_window(pkg, cuda, dtype, D, T, lens, window, sinks, beyond):
    """Keys about one block of 128 longer than the window: the last rows see the
    first keys across it.  The scores put the rows' mass on the first keys, whose
    gradients are compared by themselves: a row that is left out takes about
    (window + 128)^-1/2 of them."""
    S = window + beyond
    T = S if T is None else T
    if lens is not None:        # a whole sequence of S rows between others
        lens = [S if n == 1 else n for n in lens] if 1 in lens else lens + [S]
        T = S = sum(lens)
    q, k, v, do = _inputs(cuda, 1, T, S, 2, 1, D, dtype, seed=window + beyond)
    s0 = S - (window + beyond) if lens is not None else 0
    u = torch.nn.functional.normalize(torch.randn(D, generator=torch.Generator().manual_seed(1)), dim=0).to(cuda)
    q = (q.float() + 2 * D ** 0.25 * u).to(dtype)
    k[:, s0:s0 + sinks] = (k[:, s0:s0 + sinks].float() + 2 * D ** 0.25 * u).to(dtype)
    cu = None if lens is None else torch.tensor([0] + list(itertools.accumulate(lens)), device=cuda)
    o, lse = pkg.window_attn(q, k, v, window, sinks, cu_seqlens=cu, return_lse=True)
    _, dk, dv = pkg.window_attn_bwd(q, k, v, o, lse, do, window, sinks, cu_seqlens=cu)
    q, do = (t[0, s0:] if lens is not None else t[0] for t in (q, do))
    _, _, (_, wk, wv), (_, sk) = oracle(q, k[0, s0:], v[0, s0:], window, sinks, do=do)
    _close(dv[0, s0:s0 + sinks], wv[:sinks], 2, 0.0, "dv")
    _close(dk[0, s0:s0 + sinks], wk[:sinks], 4, sk, "dk")


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_nan_scores_of_shared_keys(pkg, cuda, D, dtype):
    """Keys of few rows, shared by workgroups: a NaN query row is NaN in o and
    lse, and so is every row over a run of keys that are all NaN; other rows keep
    their bits."""
    q, k, v, _ = _inputs(cuda, 1, 3, 4096, 2, 1, D, dtype, seed=31)
    o, lse = pkg.window_attn(q, k, v, return_lse=True)
    q2 = q.clone()
    q2[0, 1, 0, 3] = float("nan")
    o2, lse2 = pkg.window_attn(q2, k, v, return_lse=True)
    hit = torch.zeros_like(lse, dtype=torch.bool)
    hit[0, 1, 0] = True
    assert torch.isnan(o2[hit]).all() and torch.isnan(lse2[hit]).all()
    assert torch.equal(o2[~hit], o[~hit]) and torch.equal(lse2[~hit], lse[~hit])
    k2 = k.clone()
    k2[:, 512:1024] = float("nan")      # whole workgroups' shares
    o2, lse2 = pkg.window_attn(q, k2, v, return_lse=True)
    assert torch.isnan(o2).all() and torch.isnan(lse2).all()
    # rows that do not see them keep their values: the first of 3 rows ends before
    k2 = k.clone()
    k2[:, 4094] = float("nan")
    o2, lse2 = pkg.window_attn(q, k2, v, return_lse=True)
    assert torch.equal(o2[:, 0], o[:, 0]) and torch.equal(lse2[:, 0], lse[:, 0])
    assert torch.isnan(o2[:, 1:]).all() and torch.isnan(lse2[:, 1:]).all()


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("T", [1, 3])
def test_decode_nan_scores(pkg, cuda, D, dtype, T):
    """Over a cache that several workgroups share, a NaN query row, keys of a
    whole share that are NaN and an infinite value at a key of no weight are not
    lost; other rows keep their bits."""
    q, k, v, _ = _inputs(cuda, 2, T, 4096, 4, 2, D, dtype, seed=32)
    lens = torch.tensor([4096, 3000], dtype=torch.int32, device=cuda)
    o = pkg.window_attn_decode(q, k, v, lens)
    q2 = q.clone()
    q2[1, 0, 2, 3] = float("nan")
    o2 = pkg.window_attn_decode(q2, k, v, lens)
    hit = torch.zeros(o.shape[:3], dtype=torch.bool, device=cuda)
    hit[1, 0, 2] = True
    assert torch.isnan(o2[hit]).all() and torch.equal(o2[~hit], o[~hit])
    k2 = k.clone()
    k2[0, 1024:1536, 1] = float("nan")
    o2 = pkg.window_attn_decode(q, k2, v, lens)
    hit = torch.zeros_like(hit)
    hit[0, :, 2:] = True
    assert torch.isnan(o2[hit]).all() and torch.equal(o2[~hit], o[~hit])
    # scores about 400 below the rest: the weight is 0 in 32 bits, and 0 inf is NaN
    q2 = q.abs() + 1
    k2 = k.abs()
    k2[0, 1024:1536, 1] = -400.0 / D ** 0.5
    v2 = v.clone()
    v2[0, 1300, 1, 7] = float("inf")
    o2 = pkg.window_attn_decode(q2, k2, v2, lens)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, :, 2:, 7] = True
    assert not torch.isfinite(o2[hit]).any() and torch.isfinite(o2[~hit]).all()


@pytest.mark.parametrize("Hk", [1, 3])
@pytest.mark.parametrize("window,sinks", [(40, 4), (40, 150), (1, 128), (300, 20)])
@pytest.mark.parametrize("lens", [[5] * 60 + [400, 0, 0, 50, 170, 168, 167, 1, 900, 0], [700] + [2] * 70 + [168, 429],
                                  [429, 428, 427, 0, 129, 128, 168]])
def test_first_keys_of_many_sequences(pkg, cuda, lens, window, sinks, Hk):
    """Long sequences, whose later rows reach the first keys from beyond a block's
    window, among many short and empty ones; and lengths where that begins."""
    T = sum(lens)
    q, k, v, do = _inputs(cuda, 1, T, T, 2 * Hk, Hk, 64, torch.float16 if Hk == 1 else torch.bfloat16, seed=T)
    _check(pkg, q, k, v, do, window, sinks, lens=lens)


def test_fp16_gradients_of_packed_sequences_apart(pkg, cuda):
    """A sequence's gradients do not depend on its neighbours' values, nor on
    rows that no sequence holds: the same bits beside values 2^14 times as large,
    and precise by their own size."""
    lens, T = [130, 70, 200], 500
    q, k, v, do = _inputs(cuda, 1, T, T, 2, 1, 64, torch.float16, seed=41)
    cu = torch.tensor([0, 130, 200, 400], device=cuda)
    v = v * 2.0 ** -4
    v2 = v.clone()
    v2[:, 130:200] *= 2.0 ** 14
    v2[:, 400:] = 60000.0
    got = []
    for x in (v, v2):
        o, lse = pkg.window_attn(q, k, x, 50, 2, cu_seqlens=cu, return_lse=True)
        got.append(pkg.window_attn_bwd(q, k, x, o, lse, do, 50, 2, cu_seqlens=cu))
    for s, e in ((0, 130), (200, 400)):
        for a, b in zip(*got):
            assert torch.equal(a[:, s:e], b[:, s:e])
        _, _, want, sizes = oracle(q[0, s:e], k[0, s:e], v[0, s:e], 50, 2, do=do[0, s:e])
        for g, w, n, name in zip(got[1], want, (*sizes, 0.0), ("dq", "dk", "dv")):
            _close(g[0, s:e], w, 4, n, name)


def test_scale_changed_in_place(pkg, cuda):
    """A scale that comes as a tensor counts by its value at the call."""
    q, k, v, do = _inputs(cuda, 1, 100, 100, 2, 1, 64, torch.bfloat16, seed=61)
    lens = torch.tensor([100], dtype=torch.int32, device=cuda)
    scale = torch.tensor(0.1)
    for value in (0.1, 0.4):
        scale.fill_(value)
        o, lse = pkg.window_attn(q, k, v, 30, 2, scale, return_lse=True)
        want = pkg.window_attn(q, k, v, 30, 2, value, return_lse=True)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        got = pkg.window_attn_bwd(q, k, v, o, lse, do, 30, 2, scale)
        assert all(torch.equal(a, b) for a, b in zip(got, pkg.window_attn_bwd(q, k, v, o, lse, do, 30, 2, value)))
        assert torch.equal(pkg.window_attn_decode(q[:, -1:], k, v, lens, 30, 2, scale),
                           pkg.window_attn_decode(q[:, -1:], k, v, lens, 30, 2, value))
    a = q.clone().requires_grad_()
    o = pkg.window_attn(a, k, v, 30, 2, scale)
    scale.fill_(0.1)
    o.backward(do)
    assert torch.equal(a.grad, got[0])


@pytest.mark.parametrize("window,sinks", [(1, 3), (60, 0), (60, 4), (60, 130), (128, 1), (200, 33), (300, 140)])
def test_every_visible_pair_counts_once(pkg, cuda, window, sinks):
    """Scores of 0 give a row of n visible keys P = 1 / n each: with dO = n, dv of a
    key is the number of rows that see it.  Every length about the places where
    blocks, windows and segments end; fewer rows than keys; packed.  (P is within
    2^-11 of itself and n exact, so counts, of 560 at most, are within 0.28, and dv's
    rounding to 11 bits adds at most 0.25.)"""
    def check(T, S, lens=None):
        q = torch.zeros(1, T, 1, 64, dtype=torch.float16, device=cuda)
        k = torch.zeros(1, S, 1, 64, dtype=torch.float16, device=cuda)
        spans = [(0, T, 0, S)] if lens is None else \
            [(s, s + n, s, s + n) for s, n in zip(itertools.accumulate([0] + lens[:-1]), lens)]
        cu = None if lens is None else torch.tensor([0] + list(itertools.accumulate(lens)), device=cuda)
        want = torch.zeros(S, device=cuda)
        do = torch.zeros_like(q)
        for a, b, c, d in spans:
            m = visible(b - a, d - c, window, sinks, cuda)
            do[0, a:b] = m.sum(1)[:, None, None].to(do.dtype)
            want[c:d] = m.sum(0)
        o, lse = pkg.window_attn(q, k, k, window, sinks, cu_seqlens=cu, return_lse=True)
        dv = pkg.window_attn_bwd(q, k, k, o, lse, do, window, sinks, cu_seqlens=cu)[2]
        assert ((dv[0, :, 0].float() - want[:, None]).abs() <= 0.65).all(), (T, S, lens)

    for S in sorted({n for e in (window, window + 128, window + 256) for n in range(max(1, e - 2), e + 3)}):
        check(S, S)
        check(min(S, 70), S)
        check(S, S, [S])
        check(2 * S + 9, 2 * S + 9, [0, S, 7, 0, S, 2])
        check(S + 60, S + 60, [1] * 60 + [S])
