"""Rotary positions without a GPU: frequencies against their formulas, and what is refused."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from mlbricks_b200 import _ebx, rotary


def test_public_names():
    assert set(rotary.__all__) == {"SCALINGS", "frequencies", "rotate"}


@pytest.mark.parametrize("dim", [2, 6, 64, 128])
def test_frequencies(dim):
    half = dim // 2
    plain = [10000.0 ** (-2 * i / dim) for i in range(half)]
    tol = 2.0**-48  # an error of 2^-52 in the exponent, times ln 10000 < 10, and the power's own

    def same(got, want):
        assert got.dtype is torch.float64 and got.shape == (half,)
        for g, w in zip(got.tolist(), want):
            assert abs(g - w) <= tol * w

    same(rotary.frequencies(dim, device="cpu"), plain)
    same(rotary.frequencies(dim, scaling="linear", factor=4.0, device="cpu"), [f / 4 for f in plain])
    ramp = rotary.frequencies(dim, scaling="ramp", factor=8.0, trained_length=2048, device="cpu").tolist()
    for got, f in zip(ramp, plain):
        turns = 2048 * f / (2 * math.pi)
        w = f if turns >= 32 else f / 8 if turns <= 1 else f / 8 + (f - f / 8) * (turns - 1) / 31
        assert abs(got - w) <= tol * f
    based = rotary.frequencies(dim, scaling="base", factor=8.0, device="cpu").tolist()
    assert based[0] == 1.0
    if half > 1:  # the slowest pair is divided by the factor
        assert abs(based[-1] * 8 - plain[-1]) <= tol * plain[-1]


@pytest.mark.parametrize("change", [dict(rotary_dim=5), dict(rotary_dim=0), dict(scaling="other"), dict(base=-1.0),
                                    dict(factor=0.0), dict(scaling="ramp"),
                                    dict(scaling="ramp", trained_length=100, slow=3.0, fast=3.0)])
def test_frequencies_refused(change):
    with pytest.raises(ValueError):
        rotary.frequencies(**{"rotary_dim": 64, "device": "cpu", **change})


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(1, 1, 4)
    with pytest.raises(ValueError, match="CUDA"):
        rotary.rotate(x, x, torch.zeros(1, dtype=torch.int32), torch.zeros(2))


def test_argument_errors_without_gpu():
    lib = _ebx.load()

    def side(**change):
        fields = dict(input=16, output=32, in_token_stride=64, in_head_stride=64, out_token_stride=64, out_head_stride=64,
                      heads=1, reserved=0)
        return ctypes.byref(_ebx.RotarySide(*{**fields, **change}.values()))

    def call(q=None, k=None, dim=64, part=64, dtype=1, positions=8, position_bits=32, frequencies=8, frequency_bits=64,
             tokens=1, scale=1.0):
        return lib.ebx_rotate(q or side(), k, dim, part, dtype, positions, position_bits, frequencies, frequency_bits, tokens,
                              0, scale, 0, None)

    def refused(status, words):
        assert status == _ebx.EBX_ERR_INVALID
        assert words in _ebx.last_error()

    refused(lib.ebx_rotate(None, None, 64, 64, 1, 8, 32, 8, 64, 1, 0, 1.0, 0, None), "null")
    refused(call(q=side(input=None)), "null")
    refused(call(k=side(output=None)), "null")
    refused(call(positions=None), "null")
    refused(call(frequencies=None), "null")
    refused(call(part=63), "even")
    refused(call(part=66), "even")
    refused(call(part=0), "even")
    refused(call(dim=4098), "4096")
    refused(call(q=side(heads=65537)), "65536")
    refused(call(dtype=3), "dtype")
    refused(call(position_bits=16), "positions")
    refused(call(frequency_bits=16), "frequencies")
    refused(call(scale=float("inf")), "scale")
    refused(call(tokens=2**31), "tokens")
    refused(call(q=side(input=17)), "aligned")
    refused(call(q=side(heads=-1)), "heads")
    assert call(tokens=0) == _ebx.EBX_OK
    assert call(q=side(heads=0, input=None)) == _ebx.EBX_OK


def test_tensors_that_require_gradients_are_refused():
    positions, freq = torch.zeros(1, dtype=torch.int32), torch.zeros(2)
    x, g = torch.zeros(1, 1, 4), torch.zeros(1, 1, 4, requires_grad=True)
    for args in ((g, None, positions, freq), (x, g, positions, freq), (g * 2, x, positions, freq),
                 (x, None, positions, freq.clone().requires_grad_())):
        for inplace in (False, True):
            with pytest.raises(ValueError, match="backward"):
                rotary.rotate(*args, inplace=inplace)
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check
                rotary.rotate(*args, inplace=inplace)
