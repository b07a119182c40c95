"""The serving example's decoder, which trains as any module does: on the host, with gradients.

Tolerances: gradcheck's own for differences in 64 bits (steps of 1e-6: their error is some 1e-6 of the third
derivative's size from the step, and 1e-10 from rounding; it allows 1e-5 + 1e-3 of the value)."""
from __future__ import annotations

import math
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

kv_serving = pytest.importorskip("kv_serving")


def test_rotation_is_the_formula_and_its_gradient_the_turn_back():
    torch.manual_seed(0)
    dim = kv_serving.HEAD_DIM
    positions, freq = torch.tensor([0, 1, 7, 1000]), kv_serving.rotary.frequencies(dim, device="cpu")
    q, k = (torch.randn(4, h, dim, dtype=torch.float64, requires_grad=True) for h in (3, 1))
    grads = [torch.randn(4, h, dim, dtype=torch.float64) for h in (3, 1)]
    turned = kv_serving.turn(q, k, positions, freq)
    angle = positions[:, None].double() * freq
    back = torch.autograd.grad(turned, (q, k), grads)
    for x, y, g, b in zip((q, k), turned, grads, back):
        half = dim // 2
        want = torch.complex(x[..., :half], x[..., half:]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        # products and sums of 64 bits, 2^-52 of |a| + |b| each, and the angle's rounding, 2^-52 of 1000
        assert (y - torch.cat([want.real, want.imag], -1)).abs().max() < 2.0**-38
        want = torch.complex(g[..., :half], g[..., half:]) * torch.polar(torch.ones_like(angle), -angle)[:, None]
        assert (b - torch.cat([want.real, want.imag], -1)).abs().max() < 2.0**-38
    few = [torch.randn(2, h, dim, dtype=torch.float64, requires_grad=True) for h in (2, 1)]
    assert torch.autograd.gradcheck(lambda a, b: kv_serving.turn(a, b, positions[1:3], freq), few)


def test_decoder_trains_on_the_host():
    torch.manual_seed(0)
    model = kv_serving.Decoder().double()
    ids = torch.randint(kv_serving.VOCAB, (6,))
    loss = lambda: torch.nn.functional.cross_entropy(model(ids[:-1]), ids[1:])  # noqa: E731
    loss().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert all(layer.q.weight.grad.abs().max() > 0 and layer.k.weight.grad.abs().max() > 0 for layer in model.layers)
    with torch.no_grad():
        assert math.isfinite(float(loss()))
    layer = model.layers[0]
    assert layer.frequencies.dtype is torch.float64 and layer.half().frequencies.dtype is torch.float64
