"""GPU tests of cache_write_fp8, cache_read_fp8 and window_attn_decode_fp8.

Tolerances: bytes are the fp32 quotient by the stored scale, rounded to the
nearest: within half a step of e4m3 (2^-4 of the value, 2^-10 near zero) and the
quotient's own rounding.  Read back, one rounding of the product: half a step of
the type.  Attention is compared on the stored bytes, so as over a 16-bit cache:
P vs is rounded once to the operands' type before its sum, the output once behind
it, independently: within 1.5 of the type's unit (2-norm).  Scores carry k_scale in
fp32; log2 of v_scale is off by 2^-21 at most where its size is below 8, which
2^x turns into as much of P: far below a unit."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]
HALF = {**UNIT, torch.float32: 2.0 ** -24}


def _cache(dev, B, S, Hk, D, seed, spread=0.5):
    """Bytes and scales of rows of different sizes."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(B, S, Hk, D, generator=gen, device=dev) * torch.exp(
            spread * torch.randn(B, S, Hk, 1, generator=gen, device=dev))
        s = x.abs().amax(-1) / 448.0
        out += [(x / s[..., None]).to(FP8), s]
    return out[0], out[2], out[1], out[3]


def _new(dev, B, T, H, D, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(B, T, H, D, generator=gen, device=dev)).to(dtype)


# ---------------------------------------------------------------------------
# writing and reading back
# ---------------------------------------------------------------------------

def _check_written(x, cache, scale, before, scale_before, lens):
    """x [B, T, Hk, D] as the last T of lens[b] rows, everything else as before."""
    B, T = x.shape[:2]
    S = cache.shape[1]
    for b, n in enumerate(lens):
        n = min(max(n, 0), S)
        lo = max(0, n - T)
        new = x[b, T - (n - lo):].float()
        want = (new.abs().amax(-1).double() / 448.0).float()
        assert torch.equal(scale[b, lo:n], want)
        f = torch.where(want[..., None] > 0, new.double() / want[..., None].double(), 0.0)
        half = torch.clamp(f.abs() * 2.0 ** -4, min=2.0 ** -10) * (1 + 2.0 ** -20)
        assert ((cache[b, lo:n].double() - f).abs() <= half + f.abs() * 2.0 ** -22).all()
        for a, c in ((cache.view(torch.uint8), before.view(torch.uint8)), (scale, scale_before)):
            assert torch.equal(a[b, :lo], c[b, :lo]) and torch.equal(a[b, n:], c[b, n:])


@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,S,Hk,lens", [
    (1, 1, 1, 1, [1]), (3, 1, 40, 2, [1, 40, 17]), (2, 7, 50, 3, [7, 50]), (4, 5, 33, 1, [3, 0, -2, 60]),
    (2, 100, 100, 4, [100, 31]), (1, 700, 900, 2, [850])])
def test_write(pkg, cuda, dtype, D, B, T, S, Hk, lens):
    """New tokens, prompts, prompts with padding in front, lengths outside the cache."""
    kc, vc, ks, vs = _cache(cuda, B, S, Hk, D, B + T + S)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    k, v = _new(cuda, B, T, Hk, D, dtype, 1), _new(cuda, B, T, Hk, D, dtype, 2)
    k[0, -1, 0] = 0
    pkg.cache_write_fp8(k, v, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32, device=cuda))
    _check_written(k, kc, ks, before[0], before[2], lens)
    _check_written(v, vc, vs, before[1], before[3], lens)


def test_write_and_read_strides(pkg, cuda):
    """Rows as a joint product gives them, caches inside larger ones, scales with
    strides of their own, lengths of 64 bits."""
    B, T, S, Hk, D = 2, 9, 30, 2, 64
    qkv = _new(cuda, B, T, 8, D, torch.bfloat16, 3)
    _, k, v = qkv.split([4, 2, 2], 2)
    big = torch.full((2, B, S, 5, D), 0.0, device=cuda).to(FP8)
    kc, vc = big[0, :, :, 1:3], big[1, :, :, 2:4]
    scales = torch.full((Hk, 2, B, S), 7.0, device=cuda)
    ks, vs = scales[:, 0].permute(1, 2, 0), scales[:, 1].permute(1, 2, 0)
    lens = [30, 12]
    pkg.cache_write_fp8(k, v, kc, vc, ks, vs, torch.tensor(lens, device=cuda))
    zero = torch.zeros(B, S, Hk, D, device=cuda).to(FP8)
    seven = torch.full((B, S, Hk), 7.0, device=cuda)
    _check_written(k, kc, ks, zero, seven, lens)
    _check_written(v, vc, vs, zero, seven, lens)
    for part in (slice(None), slice(5, 20)):
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            got = pkg.cache_read_fp8(kc[:, part], vc[:, part], ks[:, part], vs[:, part], dtype=dtype)
            for g, c, s in zip(got, (kc, vc), (ks, vs)):
                assert g.shape == c[:, part].shape and g.dtype == dtype
                assert torch.equal(g, (c[:, part].float() * s[:, part, :, None]).to(dtype))


@pytest.mark.parametrize("D", [64, 128])
def test_read_back_of_what_was_written(pkg, cuda, D):
    B, S, Hk = 3, 77, 3
    k, v = _new(cuda, B, S, Hk, D, torch.float16, 5), _new(cuda, B, S, Hk, D, torch.float16, 6)
    kc, vc, ks, vs = _cache(cuda, B, S, Hk, D, 9)
    pkg.cache_write_fp8(k, v, kc, vc, ks, vs, torch.full((B,), S, dtype=torch.int32, device=cuda))
    for x, y in zip((k, v), pkg.cache_read_fp8(kc, vc, ks, vs, dtype=torch.float32)):
        top = x.float().abs().amax(-1, keepdim=True)
        # half a step of e4m3; at most 2^-10 of the scale near zero
        assert ((y - x.float()).abs() <= torch.maximum(x.float().abs() * 2.0 ** -4, top / 448 * 2.0 ** -10) * (1 + 2.0 ** -10)).all()


def test_rows_that_are_not_finite(pkg, cuda):
    k = _new(cuda, 1, 4, 1, 64, torch.bfloat16, 5)
    k[0, 1, 0, 3], k[0, 2, 0, 5] = float("nan"), float("inf")
    kc, vc, ks, vs = _cache(cuda, 1, 4, 1, 64, 9)
    pkg.cache_write_fp8(k, k, kc, vc, ks, vs, torch.tensor([4], dtype=torch.int32, device=cuda))
    x, _ = pkg.cache_read_fp8(kc, vc, ks, vs, dtype=torch.float32)
    assert torch.isfinite(x[0, [0, 3]]).all() and torch.isnan(x[0, 1:3]).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def oracle(q, kc, vc, ks, vs, lens, window, sinks, scale=None):
    """64 bits; masked places take part in nothing, whatever they hold."""
    B, T, Hq, D = q.shape
    S, Hk = kc.shape[1:3]
    G, scale = Hq // Hk, D ** -0.5 if scale is None else scale
    o = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        n = min(max(n, 0), S)
        for t in range(T):
            i = n - T + t
            j = torch.arange(n, device=q.device)
            j = j[(j <= i) & ((j > i - (window or S)) | (j < sinks))]
            if i < 0 or not j.numel():
                continue
            K, V = (c[b, j].double() * s[b, j].double()[..., None] for c, s in ((kc, ks), (vc, vs)))
            for h in range(Hq):
                p = torch.softmax((K[:, h // G] * q[b, t, h].double()).sum(-1) * scale, 0)
                o[b, t, h] = (p[:, None] * V[:, h // G]).sum(0)
    return o


def _close(got, want, units=1.5):
    assert torch.isfinite(got).all()
    d = (got.double() - want).norm().item()
    assert d <= units * UNIT[got.dtype] * want.norm().item() + 1e-30, d / max(want.norm().item(), 1e-30) / UNIT[got.dtype]


def _decode(pkg, q, kc, vc, ks, vs, lens, *args):
    return pkg.window_attn_decode_fp8(q, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32, device=q.device), *args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,S,Hq,Hk,window,sinks,lens", [
    (1, 1, 1, 1, 1, None, 0, [1]), (1, 1, 33, 2, 1, None, 0, [33]), (3, 1, 64, 4, 2, 7, 2, [1, 64, 20]),
    (2, 3, 100, 4, 1, 32, 0, [3, 99]), (2, 16, 90, 6, 2, 20, 5, [90, 10]), (1, 4, 700, 3, 3, None, 0, [650]),
    (2, 1, 3000, 8, 2, None, 0, [2999, 31]), (1, 2, 5000, 4, 4, 1000, 100, [4800]), (5, 1, 300, 12, 4, 64, 4, [0, 1, 64, 65, 300]),
    (1, 16, 2100, 16, 2, 300, 3, [2100]), (1, 1, 20000, 4, 1, None, 0, [19999])])
def test_decode(pkg, cuda, dtype, D, B, T, S, Hq, Hk, window, sinks, lens):
    kc, vc, ks, vs = _cache(cuda, B, S, Hk, D, B + T + S + D)
    q = _new(cuda, B, T, Hq, D, dtype, 8)
    o = _decode(pkg, q, kc, vc, ks, vs, lens, window, sinks)
    want = oracle(q, kc, vc, ks, vs, lens, window, sinks)
    _close(o, want)
    for b, n in enumerate(lens):
        hidden = max(0, T - min(max(n, 0), S))
        assert (o[b, :hidden] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [200, 4000])
def test_scales_of_all_sizes(pkg, cuda, dtype, S):
    """Rows that differ by 2^20 in size, whole caches of tiny or of zero values."""
    kc, vc, ks, vs = _cache(cuda, 2, S, 2, 128, 4)
    gen = torch.Generator(device=cuda).manual_seed(4)
    wide = torch.exp2(torch.randint(-20, 1, vs.shape, generator=gen, device=cuda).float())
    q = _new(cuda, 2, 1, 4, 128, dtype, 8)
    lens = [S, S - 70]
    for f in (wide, wide * 2.0 ** -40 if dtype == torch.bfloat16 else wide, wide * 64):
        o = _decode(pkg, q, kc, vc, ks, vs * f, lens)
        _close(o, oracle(q, kc, vc, ks, vs * f, lens, None, 0))
    assert (_decode(pkg, q, kc, vc, ks, vs * 0, lens) == 0).all()
    zeros = torch.where(torch.rand(vs.shape, generator=gen, device=cuda) < 0.5, 0.0, vs)
    _close(_decode(pkg, q, kc, vc, ks, zeros, lens), oracle(q, kc, vc, ks, zeros, lens, None, 0))
    zeros = torch.where(torch.rand(ks.shape, generator=gen, device=cuda) < 0.5, 0.0, ks)
    _close(_decode(pkg, q, kc, vc, zeros, vs, lens), oracle(q, kc, vc, zeros, vs, lens, None, 0))


@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0])
def test_scale(pkg, cuda, scale):
    kc, vc, ks, vs = _cache(cuda, 1, 90, 2, 64, 4)
    q = _new(cuda, 1, 2, 4, 64, torch.bfloat16, 8)
    _close(_decode(pkg, q, kc, vc, ks, vs, [80], None, 0, scale), oracle(q, kc, vc, ks, vs, [80], None, 0, scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [120, 2500])
def test_hidden_rows_may_hold_anything(pkg, cuda, dtype, D, S):
    """NaN bytes, NaN and infinite scales in rows that no token sees, or that only
    the later of two tokens sees."""
    kc, vc, ks, vs = _cache(cuda, 1, S, 1, D, 4)
    q = _new(cuda, 1, 3, 2, D, dtype, 8)
    n, window, sinks = S - 13, 40, 2
    want = oracle(q, kc, vc, ks, vs, [n], window, sinks)
    for rows in (slice(sinks, n - window - 2), slice(n, S)):
        for c in (kc, vc):
            c.view(torch.uint8)[:, rows] = 0x7f
        ks[:, rows], vs[:, rows] = float("nan"), float("inf")
    _close(_decode(pkg, q, kc, vc, ks, vs, [n], window, sinks), want)
    # the newest row: NaN for the last token alone
    for c, value in ((vc.view(torch.uint8), 0xff), (kc.view(torch.uint8), 0x7f), (vs, float("nan")), (ks, float("nan")),
                     (vs, float("inf"))):
        keep = c[0, n - 1].clone()
        c[0, n - 1] = value
        o = _decode(pkg, q, kc, vc, ks, vs, [n], window, sinks)
        c[0, n - 1] = keep
        assert torch.isnan(o[0, 2]).all(), value
        _close(o[:, :2], want[:, :2])
    # one NaN byte in a column of a value that everybody sees, one that the last token does not
    vc.view(torch.uint8)[0, n - 10, 0, 5] = 0x7f
    o = _decode(pkg, q, kc, vc, ks, vs, [n], window, sinks)
    cols = torch.arange(D, device=cuda) != 5
    assert torch.isnan(o[..., 5]).all()
    _close(o[..., cols], want[..., cols])
    vc.view(torch.uint8)[0, n - 10, 0, 5] = 0x20
    want = oracle(q, kc, vc, ks, vs, [n], window, sinks)
    vc.view(torch.uint8)[0, n - window - 1, 0, 5] = 0x7f        # visible to token 1 (position n - 2) no more, to token 0 it is
    o = _decode(pkg, q, kc, vc, ks, vs, [n], window, sinks)
    want2 = oracle(q, kc, vc, ks, vs, [n], window, sinks)
    assert torch.equal(torch.isnan(o.float()), torch.isnan(want2))
    _close(o[:, 2], want2[:, 2])


def test_large_scores(pkg, cuda):
    """Scores of thousands, the largest key with the smallest value."""
    kc, vc, ks, vs = _cache(cuda, 1, 500, 1, 128, 4)
    q = _new(cuda, 1, 1, 2, 128, torch.bfloat16, 8) * 30
    vs2 = torch.where(torch.arange(500, device=cuda)[None, :, None] % 3 == 0, vs * 2.0 ** -30, vs)
    _close(_decode(pkg, q, kc, vc, ks * 10, vs2, [500]), oracle(q, kc, vc, ks * 10, vs2, [500], None, 0), 2.0)


def test_strides(pkg, cuda):
    B, T, S, Hk, D = 2, 2, 60, 2, 128
    kc, vc, ks, vs = _cache(cuda, B, S, Hk, D, 4)
    big = torch.zeros(B, Hk, S + 5, 2, D, device=cuda).to(FP8)
    kc2, vc2 = (big[:, :, :S, i].transpose(1, 2) for i in range(2))
    kc2.view(torch.uint8).copy_(kc.view(torch.uint8)), vc2.view(torch.uint8).copy_(vc.view(torch.uint8))
    ks2, vs2 = ks.permute(2, 1, 0).contiguous().permute(2, 1, 0), vs.transpose(1, 2).contiguous().transpose(1, 2)
    q = _new(cuda, B, T, 8, D, torch.float16, 8)[:, :, 2:6]
    assert torch.equal(_decode(pkg, q, kc2, vc2, ks2, vs2, [60, 33], 20, 1), _decode(pkg, q.contiguous(), kc, vc, ks, vs, [60, 33], 20, 1))


def test_like_the_16_bit_cache(pkg, cuda):
    """Write, then attend, against the same through window_attn_decode on the rows
    read back: the same bytes, so only the roundings of both calls apart; the read
    rows' own rounding is one more on each of keys and values."""
    B, T, S, Hq, Hk, D = 4, 2, 600, 8, 2, 128
    k, v = _new(cuda, B, S, Hk, D, torch.bfloat16, 1), _new(cuda, B, S, Hk, D, torch.bfloat16, 2)
    kc, vc = (torch.zeros(B, S, Hk, D, device=cuda).to(FP8) for _ in range(2))
    ks, vs = torch.zeros(B, S, Hk, device=cuda), torch.zeros(B, S, Hk, device=cuda)
    lens = torch.tensor([600, 300, 599, 64], dtype=torch.int32, device=cuda)
    for t in range(2):          # the prompt, then two new tokens
        n = S - 2 if t == 0 else 2
        at = lens - 2 if t == 0 else lens
        rows = (at.long()[:, None] - n + torch.arange(n, device=cuda)).clamp(min=0)
        pick = lambda x: x.gather(1, rows[..., None, None].expand(-1, -1, Hk, D))
        pkg.cache_write_fp8(pick(k), pick(v), kc, vc, ks, vs, at)
    q = _new(cuda, B, T, Hq, D, torch.bfloat16, 3)
    got = pkg.window_attn_decode_fp8(q, kc, vc, ks, vs, lens, 128, 4)
    k16, v16 = pkg.cache_read_fp8(kc, vc, ks, vs)
    want = pkg.window_attn_decode(q, k16, v16, lens, 128, 4)
    # q k over 128 columns of relative 2^-8 errors each: scores of size 1 are off by 2^-8 about
    assert (got.double() - want.double()).norm() <= 4 * 2.0 ** -8 * want.double().norm()


def test_captured_step_with_lengths_that_grow(pkg, cuda):
    """A captured decode step (write, attend), the lengths counted up between the
    replays, against eager calls on another cache."""
    B, S, Hq, Hk, D = 3, 400, 8, 2, 64
    first, second = _cache(cuda, B, S, Hk, D, 4), [t.clone() for t in _cache(cuda, B, S, Hk, D, 4)]
    lens = torch.tensor([1, 200, 333], dtype=torch.int32, device=cuda)
    qkv = _new(cuda, B, 1, Hq + 2 * Hk, D, torch.bfloat16, 3)
    q, k, v = qkv.split([Hq, Hk, Hk], 2)

    def step(cache):
        pkg.cache_write_fp8(k, v, *cache, lens)
        return pkg.window_attn_decode_fp8(q, *cache, lens, 100, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(second)
        step(first)         # (capturing does not run it)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(first)
    for i in range(4):
        lens += 1
        qkv.copy_(_new(cuda, B, 1, Hq + 2 * Hk, D, torch.bfloat16, 10 + i))
        graph.replay()
        want = step(second)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_fixed_order(pkg, cuda):
    kc, vc, ks, vs = _cache(cuda, 2, 9000, 2, 128, 4)
    q = _new(cuda, 2, 1, 8, 128, torch.float16, 8)
    runs = [_decode(pkg, q, kc, vc, ks, vs, [9000, 5000]) for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_offsets_beyond_32_bits(pkg, cuda):
    """Caches of more than 2^31 bytes: written, read back and attended at their end."""
    B, S, Hk, D, Hq = 2, 33_000, 256, 128, 512
    kc, vc = (torch.zeros(B, S, Hk, D, dtype=torch.uint8, device=cuda).view(FP8) for _ in range(2))
    ks, vs = torch.zeros(B, S, Hk, device=cuda), torch.zeros(B, S, Hk, device=cuda)
    lens = torch.tensor([S, S - 11], dtype=torch.int32, device=cuda)
    k, v = _new(cuda, B, 40, Hk, D, torch.bfloat16, 1), _new(cuda, B, 40, Hk, D, torch.bfloat16, 2)
    pkg.cache_write_fp8(k, v, kc, vc, ks, vs, lens)
    q = _new(cuda, B, 1, Hq, D, torch.bfloat16, 3)
    o = pkg.window_attn_decode_fp8(q, kc, vc, ks, vs, lens, 30)
    tail = slice(S - 60, S)
    _check_written(k, kc[:, tail], ks[:, tail], torch.zeros_like(kc[:, tail], dtype=torch.uint8).view(FP8),
                   torch.zeros_like(ks[:, tail]), [60, 49])
    assert (ks[:, :S - 60] == 0).all()
    _close(o, oracle(q, kc[:, tail], vc[:, tail], ks[:, tail], vs[:, tail], [60, 49], 30, 0))
    k16, _ = pkg.cache_read_fp8(kc, vc, ks, vs)
    assert torch.equal(k16[:, tail], (kc[:, tail].float() * ks[:, tail, :, None]).bfloat16())
