"""The angles of rotary positions, to the last bits of 32: what is left when a reduced angle is rounded to 32 bits counts too.

Pairs (1, 0) give the cosine and the sine themselves.  Tolerance, from the arithmetic: an angle of h + r half turns has h in 32
bits and r, at most 2^-25, apart.  CUDA's sine and cosine of h half turns are off by 2 units of their last place at
most, 2^-22 of the value s' at h, and |s'| <= |s| + 2^-23; pi r times the other one adds what r stands for, with errors
of 2^-46 from each of its factors and 2^-47 from the next term of the series; the sum is rounded by half a unit, 2^-24 |s|.
The angle has 64 bits: the frequency times the position, 1 / (2 pi), and their product, and in the formula once more, make less
than 2^-50 of it.  Together (2.5 2^-23) (|s| + 2^-23) + 2^-44 + 2^-50 angle.

That is far less than what dropping r changes, up to pi 2^-25, wherever s is small; the test says so of the formula."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

rotary = pytest.importorskip("mlbricks_b200.rotary")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("places", [64, 10_000, 1_000_000])
def test_sines_keep_what_32_bits_leave(cuda_ok, interleaved, places):
    torch.manual_seed(places)
    tokens, dim = 2000, 128
    positions, freq = torch.randint(-places, places, (tokens,), device="cuda"), rotary.frequencies(dim)
    x = torch.zeros(tokens, 1, dim, device="cuda")
    first = slice(0, dim, 2) if interleaved else slice(0, dim // 2)
    second = slice(1, dim, 2) if interleaved else slice(dim // 2, dim)
    x[..., first] = 1
    y, _ = rotary.rotate(x, None, positions, freq, interleaved=interleaved)

    angle = positions.double()[:, None] * freq
    half_turns = angle / math.pi
    half_turns = half_turns - 2 * torch.round(half_turns / 2)
    rounded = half_turns.float().double()
    for got, of, slope in ((y[:, 0, first], torch.cos, lambda t: -torch.sin(t)), (y[:, 0, second], torch.sin, torch.cos)):
        want = of(angle)
        tol = 2.5 * 2.0**-23 * (want.abs() + 2.0**-23) + 2.0**-44 + 2.0**-50 * angle.abs()
        assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max()
        # the formula without the rest, and with the rest the wrong way round, would be noticed
        dropped = of(math.pi * rounded)
        wrong = dropped - math.pi * (half_turns - rounded) * slope(math.pi * rounded)
        assert ((dropped - want).abs() > tol).sum() > 1000 and ((wrong - want).abs() > tol).sum() > 1000
