"""GPU tests of the quantisers at their largest sizes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


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
