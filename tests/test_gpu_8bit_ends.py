"""GPU tests of the quantisers at their largest sizes."""

import pytest
import torch

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
