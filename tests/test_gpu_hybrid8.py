"""GPU tests of the hybrid model's loss and of its 8-bit form: the run of
linear_xent, quantize_fp8, fp8_linear and the 8-bit cache together."""

import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_model.py")


@pytest.fixture(scope="module")
def hybrid():
    spec = importlib.util.spec_from_file_location("hybrid_model", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_gradients_of_the_loss(hybrid, cuda):
    """model.loss against the cross entropy of the model's rows in 64 bits, with
    padding: the head's gradient and, by the rows', every other parameter's start."""
    torch.manual_seed(0)
    model = hybrid.HybridModel(layers=1).to(cuda)
    t = hybrid.text(3, 71, 64, 1, cuda)
    tokens, targets = t[:, :-1], t[:, 1:].clone()
    targets[1, 40:] = -1
    rows = model.rows(tokens)
    rows.retain_grad()
    losses = hybrid.gdn.linear_xent(rows, model.head.weight, targets)
    loss = losses.sum() / (targets >= 0).sum()
    loss.backward()
    assert torch.equal(loss, model.loss(tokens, targets))
    x = rows.detach().double().requires_grad_()
    w = model.head.weight.detach().double().requires_grad_()
    want = F.cross_entropy((x @ w.T).flatten(0, 1), targets.flatten(), ignore_index=-1)
    want.backward()
    assert abs(loss.item() - want.item()) <= 2.0 ** -15 * (1 + want.item())
    # one rounding of the probabilities and one of the result
    for got, ref in ((rows.grad, x.grad), (model.head.weight.grad, w.grad)):
        assert (got.double() - ref).norm() <= 1.5 * 2.0 ** -8 * ref.norm()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


def test_answer_in_8_bits(hybrid, cuda):
    """Prompts in pieces, then token by token, against one token at a time: the same
    bytes in the cache and the same 8-bit operands but for the roundings to 16 bits
    on the way (as between the two ways of the 16-bit model), which can move an
    e4m3 operand by a whole step, 2^-3, where they pass a border of rounding: a
    share 2^-8 / 2^-3 of the operands does, each by 2^-3 of its size, so a product is
    off by (2^-5)^0.5 2^-3 = 2^-5.5 at most; 6 mixers of two products in a row and the
    head's, independent, add to 13^0.5 2^-5.5."""
    torch.manual_seed(1)
    model = hybrid.to_8_bits(hybrid.HybridModel().to(cuda))
    tokens = hybrid.text(3, 130, 64, 5, cuda)
    out, got = hybrid.answer_8_bits(model, tokens, 3)
    assert torch.equal(out[:, :130], tokens) and out.shape == (3, 133) and got.shape == (3, 132, 64)
    _, want = hybrid.answer_8_bits(model, tokens, 3, piece=1)
    assert torch.isfinite(got).all()
    err = ((got[:, :130] - want[:, :130]).norm() / want[:, :130].norm()).item()
    assert err <= 13 ** 0.5 * 2.0 ** -5.5, err


def test_8_bits_against_16(hybrid, cuda):
    """Every product has two e4m3 operands, each off by a relative 2^-4 at most, on
    average (evenly spread) 2^-4 / 3^0.5: 2^0.5 of that a product; two products a
    mixer, 6 of them, the head's, and the attention's keys and values (one more of
    each), independent."""
    torch.manual_seed(1)
    model = hybrid.HybridModel().to(cuda)
    tokens = hybrid.text(3, 100, 64, 5, cuda)
    with torch.no_grad():
        want = model(tokens)
    _, got = hybrid.answer_8_bits(hybrid.to_8_bits(model), tokens, 1)
    err = ((got[:, :100] - want).norm() / want.norm()).item()
    assert err <= (13 + 2) ** 0.5 * 2.0 ** -4 * (2.0 / 3.0) ** 0.5, err
