"""CPU tests of the sizes that linear_xent, the 8-bit product and the 8-bit cache take,
at their ends (nothing is enqueued: what is in order but for its workspace is told so),
and of further refusals."""

import ctypes
import importlib.util
import os

import pytest
import torch
from test_head_and_fp8_host import _operands, _xent, lib  # noqa: F401


@pytest.mark.parametrize("name", ["gdn_xent", "gdn_xent_bwd"])
@pytest.mark.parametrize("kw,ok", [
    (dict(N=1_000_000, V=151_936), True), (dict(N=4_000_000, V=128_000), True), (dict(N=(1 << 26) - 1, V=7900), True), (dict(N=(1 << 26) - 1, V=8000), False),
    (dict(N=40, V=1 << 28), True), (dict(N=5_000_000, V=128_000), False), (dict(N=1 << 20, V=1 << 20), False)])
def test_xent_takes_what_a_launch_holds(lib, pkg, name, kw, ok):  # noqa: F811
    P = lambda **more: ctypes.byref(_xent(pkg._lib, **kw, **more))
    assert getattr(lib, name + "_launch")(P(workspace=None), None) == (1006 if ok else 1002)
    assert (getattr(lib, name + "_workspace_size")(P()) > 0) == ok


def test_too_many_logits_is_a_value_error(pkg, monkeypatch):
    from importlib import import_module
    L = import_module("v100-attention-lab_amd.loss")
    monkeypatch.setattr(L, "_validate", lambda *a: None)
    x, w = (torch.empty(1, 64, dtype=torch.float16).expand(n, 64) for n in (1 << 20, 1 << 20))
    with pytest.raises(ValueError, match="does not support"):
        L._plan(x, w, None, None, None, False)


def test_xent_workspace_is_what_the_tiles_leave(lib, pkg):  # noqa: F811
    """A pair (8 bytes) for a row and tile of the vocabulary, 256 words in the large
    tiles and 128 in the others, and a row's target logit."""
    size = lambda **kw: lib.gdn_xent_workspace_size(ctypes.byref(_xent(pkg._lib, **kw)))
    assert size(N=1_000_000, V=128_000) == 1_000_000 * (500 * 8 + 4)
    assert size(N=8192, V=32_001) == 8192 * (126 * 8 + 4)
    assert size(N=64, V=50_257) == 64 * (393 * 8 + 4)
    assert size(N=1000, V=500) == 1000 * (4 * 8 + 4)


@pytest.mark.parametrize("i", [0, 1])
def test_scales_with_a_gradient_are_not_written(pkg, i):
    """They would change under the graph that holds them."""
    o = _operands()
    scales = [o["ks"].clone(), o["ks"].clone()]
    scales[i].requires_grad_()
    write = lambda: pkg.cache_write_fp8(o["k"], o["k"], o["kc"], o["kc"], *scales, o["lens"])
    with pytest.raises(NotImplementedError, match="no gradient"):
        write()
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        write()


def test_a_piece_without_its_length_is_refused(pkg):
    """The hybrid model in 8 bits reads back as many rows as it is told; nothing is
    counted up before."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_model.py")
    spec = importlib.util.spec_from_file_location("hybrid_model", path)
    hybrid = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(hybrid)
    m = hybrid.WindowAttention(256, 4, 2, 64, 48, 4)
    m.eight = True
    state = m.start(1, 40, "cpu")
    with torch.no_grad(), pytest.raises(ValueError, match="length"):
        m(torch.zeros(1, 17, 256, dtype=torch.bfloat16), state)
    assert state[-1].tolist() == [0]
