"""GPU tests of the hybrid model of examples/: it learns, and answering token by
token from its states and caches gives the logits of the whole sequence."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_model.py")


@pytest.fixture(scope="module")
def hybrid():
    spec = importlib.util.spec_from_file_location("hybrid_model", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_learns(hybrid, cuda):
    torch.manual_seed(0)
    model = hybrid.HybridModel(layers=1).to(cuda)
    losses = hybrid.train(model, 30, batch=4, length=200)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5])


@pytest.mark.parametrize("fp8", [False, True])
def test_token_by_token(hybrid, cuda, fp8):
    """The two ways round at different places: 6 mixers of about 6 roundings to
    bf16 each in a row are within 6 * 2^-8 of the logits' size; the 8-bit norms
    (relative step 2^-4) replace those of 7 norms, half a step each, independent:
    7^0.5 * 2^-5."""
    torch.manual_seed(1)
    model = hybrid.HybridModel().to(cuda)
    tokens = hybrid.text(3, 130, 64, 5, cuda)
    with torch.no_grad():
        want = model(tokens)
    all_tokens, got = hybrid.answer(model, tokens, 2, fp8)
    assert torch.equal(all_tokens[:, :130], tokens) and all_tokens.shape == (3, 132)
    err = ((got[:, :130] - want).norm() / want.norm()).item()
    assert err <= 6 * 2.0 ** -8 + (7 ** 0.5 * 2.0 ** -5 if fp8 else 0.0)
