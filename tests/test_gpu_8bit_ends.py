"""GPU tests of the quantisers and of the 8-bit cache at their largest sizes, of the
cache at the smallest values and of the 8-bit product where its terms cancel."""

import pytest
import torch
from test_gpu_cache8 import FP8, _decode, _new, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [128, None])
def test_more_rows_than_a_launch_holds(pkg, cuda, group):
    """2^24 rows and more, a workgroup each; only the last ones hold anything."""
    rows = 2 ** 24 + 1000
    x = torch.zeros(rows, 128, dtype=torch.bfloat16, device=cuda)
    at = torch.cat([torch.arange(2 ** 23 - 50, 2 ** 23 + 50, device=cuda), torch.arange(rows - 100, rows, device=cuda)])
    x[at] = torch.randn(200, 128, device=cuda).bfloat16()
    q, s = pkg.quantize_fp8(x, group=group)
    q2, s2 = pkg.quantize_fp8(x[at], group=group)
    assert torch.equal(q.view(torch.uint8)[at], q2.view(torch.uint8)) and torch.equal(s[at], s2) and (s2 > 0).all()
    assert int((s != 0).sum()) == 200


@pytest.mark.parametrize("form", ["groups", "row", "blocks"])
def test_the_longest_row(pkg, cuda, form):
    """2^31 - 128 columns: what counts past the last one is no negative number."""
    D = 2 ** 31 - 128
    x = torch.zeros(1, D, dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    x[0, -300:] = torch.randn(300, generator=gen, device=cuda).bfloat16()
    quantize = {"groups": pkg.quantize_fp8, "row": lambda z: pkg.quantize_fp8(z, group=None),
                "blocks": pkg.quantize_fp8_weight}[form]
    q, s = quantize(x)
    q2, s2 = quantize(x[:, -384:].contiguous())
    assert torch.equal(q.view(torch.uint8)[:, -384:], q2.view(torch.uint8)) and torch.equal(s[:, -s2.shape[1]:], s2)
    assert int((q.view(torch.uint8)[:, :-300] != 0).any()) == 0
    assert int((s != 0).sum()) == s2.shape[1]


def _all_rows_are(t, row):
    """t [rows, n bytes] holds `row` everywhere."""
    words, row = t.view(torch.int64), row.view(torch.int64)
    for i in range(0, len(words), 2 ** 25):
        assert bool((words[i:i + 2 ** 25] == row).all()), i


def test_a_prompt_of_more_rows_than_a_launch_holds(pkg, cuda):
    """2^28 rows and more are 2^32 threads for keys and values; the rows behind are left."""
    T, D = 2 ** 28 + 7, 128
    gen = torch.Generator(device=cuda).manual_seed(1)
    k, v = torch.randn(2, 1, 1, 1, D, generator=gen, device=cuda).bfloat16().unbind()
    kc, vc = (torch.zeros(1, T + 9, 1, D, dtype=torch.uint8, device=cuda).view(FP8) for _ in range(2))
    ks, vs = torch.zeros(1, T + 9, 1, device=cuda), torch.zeros(1, T + 9, 1, device=cuda)
    lens = torch.tensor([T], dtype=torch.int32, device=cuda)
    pkg.cache_write_fp8(k.expand(1, T, 1, D), v.expand(1, T, 1, D), kc, vc, ks, vs, lens)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        q, scale = pkg.quantize_fp8(x.view(1, D), group=None)
        _all_rows_are(c.view(torch.uint8)[0, :T, 0], q.view(torch.uint8))
        assert bool((s[0, :T] == scale).all()) and not s[0, T:].any() and not c.view(torch.uint8)[0, T:].any()


def test_a_cache_of_more_rows_than_a_launch_holds(pkg, cuda):
    S, D = 2 ** 28 + 7, 128
    gen = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(2, D, generator=gen, device=cuda).to(FP8).view(torch.uint8)
    kc, vc = q.view(FP8).view(2, 1, 1, 1, D).expand(2, 1, S, 1, D).unbind()
    ks, vs = torch.tensor([0.5, 2.0], device=cuda).view(2, 1, 1, 1).expand(2, 1, S, 1).unbind()
    for x, row, f in zip(pkg.cache_read_fp8(kc, vc, ks, vs), q.view(FP8), (0.5, 2.0)):
        _all_rows_are(x.view(S, D), (row.float() * f).bfloat16())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [100, 3000])
def test_values_near_the_smallest_numbers(pkg, cuda, D, S):
    """Values of 2^-121, whose scale is no normal number any more: the output is of the
    values' own size and off by the roundings of P vs and of itself, 1.5 units, alone
    (log2 of the scale, about 128, by 2^-17)."""
    k, v = _new(cuda, 1, S, 2, D, torch.bfloat16, 1), _new(cuda, 1, S, 2, D, torch.bfloat16, 2) * 2.0 ** -121
    kc, vc = (torch.zeros(1, S, 2, D, device=cuda).to(FP8) for _ in range(2))
    ks, vs = torch.zeros(1, S, 2, device=cuda), torch.zeros(1, S, 2, device=cuda)
    pkg.cache_write_fp8(k, v, kc, vc, ks, vs, torch.tensor([S], dtype=torch.int32, device=cuda))
    q = _new(cuda, 1, 1, 4, D, torch.bfloat16, 3) * 4
    o = _decode(pkg, q, kc, vc, ks, vs, [S]).double() * 2.0 ** 121
    want = oracle(q, kc, vc, ks, vs, [S], None, 0) * 2.0 ** 121
    assert 0 < vs.max().item() < 2.0 ** -126
    assert ((o - want).norm() / want.norm()).item() <= 1.5 * 2.0 ** -8


@pytest.mark.parametrize("M", [1, 40, 700])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
def test_terms_that_cancel(pkg, cuda, M, out):
    """448 and -448 side by side, small numbers between them: fp32 sums are off by
    (K + K / 128) 2^-24 of the terms' sizes at most, 16-bit results come from products
    cut at 2^-13 of the largest of 8, 2^-10 of the terms' sizes, and are rounded."""
    K, N = 512, 300
    gen = torch.Generator(device=cuda).manual_seed(M)
    x = torch.randn(M, K, generator=gen, device=cuda)
    x[:, 0::4], x[:, 1::4] = 448.0, -448.0
    x, w = x.to(FP8), torch.randn(N, K, generator=gen, device=cuda)
    w[:, 1::4] = w[:, 0::4]
    w = w.to(FP8)
    xs, ws = torch.full((M, K // 128), 0.25, device=cuda), torch.full((-(-N // 128), K // 128), 0.5, device=cuda)
    y = pkg.fp8_linear(x, xs, w, ws, out_dtype=out)
    a, b = x.double() / 4, w.double() / 2
    want, size = a @ b.T, a.abs() @ b.abs().T
    assert (want.abs().mean() < 2.0 ** -8 * size.mean()).item()
    half = torch.finfo(out).eps / 2
    bound = size * ((K + K // 128) * 2.0 ** -24 + (0.0 if out == torch.float32 else 2.0 ** -10)) * (1 + half) + half * want.abs()
    assert ((y.double() - want).abs() / bound).max().item() <= 1
