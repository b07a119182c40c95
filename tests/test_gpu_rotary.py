"""Rotary positions against the formula in 64 bits.

Tolerance, from the arithmetic: an angle in turns is reduced in 64 bits (2^-52 of its size) and rounded to
32 bits at half a turn at most, so it is off by 2 pi 2^-26 < 2^-23; sine and cosine add 2 units of the last place
of a value up to 1, 2^-22; times the scale, the two products and their sum add 3 2^-24 of what they add up.
Together less than 2^-21 scale (|a| + |b|), and the output's own rounding: half a step of its type.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

rotary = pytest.importorskip("mlbricks_b200.rotary")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def want(x, positions, freq, interleaved, scale):
    """The turned x, and the sizes that its error goes by, in 64 bits."""
    part = 2 * freq.numel()
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    angle = positions.double()[:, None, None] * freq.double()
    a, b = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    u, v = x[..., a].double(), x[..., b].double()
    y[..., a] = scale * (u * angle.cos() - v * angle.sin())
    y[..., b] = scale * (v * angle.cos() + u * angle.sin())
    size[..., a] = size[..., b] = abs(scale) * (u.abs() + v.abs())
    return y, size


def check(x, got, positions, freq, interleaved=False, scale=1.0):
    y, size = want(x, positions, freq, interleaved, scale)
    half_step = torch.finfo(x.dtype).eps / 2
    least = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}[x.dtype]  # half the least subnormal
    # 2^-51: the angle's own rounding, in the formula and in the kernel
    turn = 2.0**-51 * (positions.double().abs()[:, None, None] * freq.double().max() + 1)
    err = 2.0**-21 * size + turn * size
    tol = err + half_step * (y.abs() + err) + least
    assert got.shape == x.shape and got.dtype is x.dtype
    assert ((got.double() - y).abs() <= tol).all(), ((got.double() - y).abs() / tol).max()
    part = 2 * freq.numel()
    assert torch.equal(got[..., part:], x[..., part:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim, part", [(32, 32), (128, 128), (128, 64), (80, 52), (96, 24), (5, 4), (2, 2), (256, 256), (66, 34),
                                       (64, 2), (40, 40)])
def test_formula(dtype, interleaved, dim, part):
    for tokens, heads, kv in ((1, 1, 1), (7, 12, 1), (133, 5, 2)):
        fused = (2 * torch.randn(tokens, heads + 2 * kv, dim, device="cuda")).to(dtype)
        q, k = fused[:, :heads], fused[:, heads:heads + kv]
        positions = torch.randint(0, 131072, (tokens,), dtype=torch.int32, device="cuda")
        positions[0] = 0
        freq = rotary.frequencies(part)
        a, b = rotary.rotate(q, k, positions, freq, interleaved=interleaved)
        check(q, a, positions, freq, interleaved)
        check(k, b, positions, freq, interleaved)
        assert torch.equal(a[0], q[0]) and torch.equal(b[0], k[0])  # position 0


@pytest.mark.parametrize("tokens, heads, kv", [(1, 64, 8), (3, 1, 1), (2049, 12, 1), (6001, 32, 8), (20011, 3, 1)])
def test_sizes(tokens, heads, kv):
    q, k = (torch.randn(tokens, h, 64, device="cuda").half() for h in (heads, kv))
    positions = torch.arange(tokens, dtype=torch.int64, device="cuda") + 1000
    freq = rotary.frequencies(64)
    a, b = rotary.rotate(q, k, positions, freq)
    check(q, a, positions, freq)
    check(k, b, positions, freq)


def test_far_and_negative_positions_and_scale():
    for dtype in (torch.int32, torch.int64):
        positions = torch.tensor([0, 1, -1, 2**31 - 1, -2**31, 10**6, 12345, -999983], dtype=dtype, device="cuda")
        if dtype is torch.int64:
            positions[3] = 2**40 + 1
        q = torch.randn(8, 4, 32, device="cuda")
        for freq in (rotary.frequencies(32), rotary.frequencies(32).float(), rotary.frequencies(32, scaling="linear", factor=3.0)):
            a, none = rotary.rotate(q, None, positions, freq, scale=-1.25)
            assert none is None
            check(q, a, positions, freq, scale=-1.25)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("part", [32, 64, 20])
def test_in_place(interleaved, part):
    fused = torch.randn(37, 9, 64, device="cuda").half()
    before = fused.clone()
    positions, freq = torch.arange(37, dtype=torch.int32, device="cuda"), rotary.frequencies(part)
    q, k = fused[:, :6], fused[:, 6:8]
    a, b = rotary.rotate(q, k, positions, freq, interleaved=interleaved, inplace=True)
    assert a is q and b is k
    c, d = rotary.rotate(before[:, :6], before[:, 6:8], positions, freq, interleaved=interleaved)
    assert torch.equal(q, c) and torch.equal(k, d) and torch.equal(fused[:, 8], before[:, 8])


def test_strides():
    positions, freq = torch.arange(11, dtype=torch.int32, device="cuda"), rotary.frequencies(32)
    base = torch.randn(11 * 5 * 40 + 7, device="cuda").half()
    odd = base[1:1 + 11 * 5 * 33].view(11, 5, 33)[..., :32]  # odd strides, a base of 2 bytes
    flat = torch.randn(5, 11, 32, device="cuda").half().transpose(0, 1)  # heads outermost
    last = torch.randn(11, 32, 5, device="cuda").half().transpose(1, 2)  # the last dimension is not contiguous
    wide = torch.randn(11, 1, 32, device="cuda").half().expand(11, 5, 32)
    for x in (odd, flat, last, wide):
        a, b = rotary.rotate(x, x, positions, freq)
        check(x, a, positions, freq)
        assert torch.equal(a, b)
    for x in (last, wide):
        with pytest.raises(ValueError, match="in place"):
            rotary.rotate(x, None, positions, freq, inplace=True)
    for x in (odd, flat):
        y, _ = rotary.rotate(x, None, positions, freq)
        rotary.rotate(x, None, positions, freq, inplace=True)
        assert torch.equal(x, y)


def test_values_that_are_not_finite():
    q = torch.randn(3, 2, 32, device="cuda").half()
    q[1, 0, 3], q[1, 1, 4], q[2, 0, 0] = math.inf, math.nan, -math.inf
    positions, freq = torch.tensor([5, 6, 0], dtype=torch.int32, device="cuda"), rotary.frequencies(32)
    a, _ = rotary.rotate(q, None, positions, freq)
    clean = torch.isfinite(q)
    pair = clean & clean.roll(16, -1)
    fresh = torch.where(clean, q, 0)
    b, _ = rotary.rotate(fresh, None, positions, freq)
    assert torch.equal(a[pair], b[pair]) and not torch.isfinite(a[~clean]).any()


def test_nothing_to_do_and_refusals():
    positions, freq = torch.zeros(0, dtype=torch.int32, device="cuda"), rotary.frequencies(32)
    a, b = rotary.rotate(torch.zeros(0, 3, 32, device="cuda"), torch.zeros(0, 1, 32, device="cuda"), positions, freq)
    assert a.shape == (0, 3, 32) and b.shape == (0, 1, 32)
    x, p = torch.zeros(4, 2, 32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for args, words in [((x.double(), None, p, freq), "float32"), ((x, x.half(), p, freq), "same dtype"),
                        ((x, x[:3], p, freq), "same tokens"), ((x, None, p[:3], freq), "positions"),
                        ((x, None, p.float(), freq), "positions"), ((x, None, p, freq.half()), "frequencies"),
                        ((x, None, p, rotary.frequencies(34)), "half of"), ((x, None, p, freq[:0]), "half of"),
                        ((x[0], None, p, freq), "q and k must be"), ((x, None, p.cpu(), freq), "positions"),
                        ((x, None, p.repeat(2)[::2], freq), "positions")]:
        with pytest.raises(ValueError, match=words):
            rotary.rotate(*args)
    with pytest.raises(ValueError, match="same memory"):
        rotary.rotate(x, x, p, freq, inplace=True)


def test_other_stream_and_graph():
    q = torch.randn(64, 8, 128, device="cuda").half()
    positions, freq = torch.arange(64, dtype=torch.int32, device="cuda"), rotary.frequencies(128)
    plain, _ = rotary.rotate(q, None, positions, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = rotary.rotate(q, None, positions, freq)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(plain, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, _ = rotary.rotate(q, None, positions, freq)
    q.copy_(torch.randn(64, 8, 128, device="cuda").half())
    positions.add_(100)
    graph.replay()
    fresh, _ = rotary.rotate(q, None, positions, freq)
    assert torch.equal(held, fresh)


def test_offsets_past_32_bits():
    """More than 2^32 bytes and 2^31 elements: the last tokens as well as the first."""
    tokens, heads, dim = 70001, 64, 512
    q = torch.empty(tokens, heads, dim, dtype=torch.float16, device="cuda")
    q[:3], q[-3:] = torch.randn(3, heads, dim, device="cuda").half(), torch.randn(3, heads, dim, device="cuda").half()
    assert q.numel() > 2**31
    positions, freq = torch.arange(tokens, dtype=torch.int32, device="cuda"), rotary.frequencies(dim)
    ends = torch.tensor([0, 1, 2, tokens - 3, tokens - 2, tokens - 1], device="cuda")
    before = q[ends].clone()
    rotary.rotate(q, None, positions, freq, inplace=True)
    check(before, q[ends], positions[ends], freq)
