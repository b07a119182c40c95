"""Rotation next to autograd: it has no backward pass, and says so instead of giving wrong gradients."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

rotary = pytest.importorskip("mlbricks_b200.rotary")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def test_gradients_are_refused_where_they_are_recorded():
    positions, freq = torch.arange(5, dtype=torch.int32, device="cuda"), rotary.frequencies(32)
    x = torch.randn(5, 2, 32, device="cuda")
    g = x.clone().requires_grad_()
    for q, k in ((g, None), (x, g), (g * 2, x)):
        with pytest.raises(ValueError, match="backward"):
            rotary.rotate(q, k, positions, freq)
    y = g * 1
    with pytest.raises(ValueError, match="backward"):
        rotary.rotate(y, None, positions, freq, inplace=True)
    assert torch.equal(y, x)
    want, _ = rotary.rotate(x, None, positions, freq)
    for how in (torch.no_grad, torch.inference_mode):
        with how():
            got, _ = rotary.rotate(g, None, positions, freq)
            assert torch.equal(got, want)
            turned = g * 1
            rotary.rotate(turned, None, positions, freq, inplace=True)
            assert torch.equal(turned, want)
    got, _ = rotary.rotate(x, None, positions, freq)  # nothing requires gradients
    assert torch.equal(got, want)


@pytest.mark.parametrize("which", ["q", "k"])
def test_a_saved_tensor_that_is_turned_in_place_is_noticed(which):
    positions, freq = torch.arange(5, dtype=torch.int32, device="cuda"), rotary.frequencies(32)
    fused = torch.randn(5, 3, 32, device="cuda")
    q, k = fused[:, :2], fused[:, 2:]
    weight = torch.ones((), device="cuda", requires_grad=True)
    loss = (weight * (q if which == "q" else k)).sum()  # saves it
    rotary.rotate(q, k, positions, freq)
    loss.backward(retain_graph=True)
    if which == "q":
        rotary.rotate(q, None, positions, freq, inplace=True)
    else:
        rotary.rotate(torch.zeros(5, 2, 32, device="cuda"), k, positions, freq, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
