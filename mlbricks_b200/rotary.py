"""Rotary positions of queries and keys (``libebx``, include/ebx.h ``ebx_rotate``).

``rotate`` turns pairs of a head's elements by angles that grow with the token's position, in one launch
for queries and keys: half and interleaved pairs, a part of the head, positions as
``mlbricks_b200.kvcache.plan`` gives them.  ``frequencies`` gives the pairs' frequencies, scaled for
contexts longer than those that a model was trained on.  Inference only, as the rest of the native route: there is no
backward pass, and where one is being recorded ``rotate`` refuses tensors that require gradients.  The reference
has no counterpart.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _ebx
from .kvcache import _DTYPES, _stream

SCALINGS = ("none", "linear", "base", "ramp")


def frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                trained_length: int = 0, slow: float = 1.0, fast: float = 32.0, device="cuda") -> torch.Tensor:
    """Angles [rotary_dim / 2] (float64) of the pairs at position 1: base ** (-2 i / rotary_dim), and for
    contexts ``factor`` times as long as trained

    * ``"linear"``: all divided by ``factor``;
    * ``"base"``: a larger base, with which the slowest pair is divided by ``factor`` and the fastest kept;
    * ``"ramp"``: pairs that make ``slow`` turns or fewer within ``trained_length`` are divided by
      ``factor``, those that make ``fast`` or more are kept, and those between go from one to the other linearly in their
      number of turns.

    The bounds of a ramp are part of what a model was trained with: give both as its configuration has them.  Configurations
    whose ramp is linear in turns usually have ``slow=1, fast=4``.  Others, often with 1 and 32, mean a ramp that is linear in the
    pair's index between the pairs that make so many turns: another formula, which this is not, with these numbers or any."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (base > 0 and math.isfinite(base) and factor > 0 and math.isfinite(factor)):
        raise ValueError("base and factor must be positive and finite")
    half = rotary_dim // 2
    if scaling == "base" and half > 1:
        base = base * factor ** (half / (half - 1))
    freq = base ** (-torch.arange(half, dtype=torch.float64) / half)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":
        if trained_length <= 0 or not fast > slow:
            raise ValueError("a ramp needs trained_length > 0 and fast > slow")
        turns = trained_length * freq / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freq = freq / factor * (1 - keep) + freq * keep
    return freq.to(device)


def _apart(x: torch.Tensor) -> bool:
    """No two elements of x at one place."""
    room = 1
    for stride, size in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if stride < room:
            return False
        room = stride * (size - 1) + room
    return True


def rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *,
           interleaved: bool = False, scale: float = 1.0, inplace: bool = False):
    """Queries [tokens, heads, head_dim] and keys [tokens, kv_heads, head_dim] (fp16, bf16 or fp32, any
    strides) turned by ``positions`` [tokens] (int32 or int64, any sign) times ``frequencies``
    [rotary_dim / 2] (float64 or float32).  Pair i is elements (i, rotary_dim / 2 + i) of a head, or (2 i, 2 i + 1) if
    ``interleaved``; elements from rotary_dim on stay as they are.  ``scale`` multiplies what was turned.

    Returns (q, k) as new tensors, or, ``inplace``, the same tensors turned where they are (their
    last dimension is then contiguous, and they share no elements).  ``k`` may be None."""
    dtype, device, shape = q.dtype, q.get_device(), q.shape
    if torch.is_grad_enabled() and (q.requires_grad or frequencies.requires_grad or (k is not None and k.requires_grad)):
        raise ValueError("rotate has no backward pass: call it under torch.no_grad(), or with detached tensors")
    if device < 0:
        raise ValueError("rotate needs CUDA tensors")
    if dtype not in _DTYPES:
        raise ValueError("q must be float32, float16 or bfloat16")
    if len(shape) != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != shape[0] or k.shape[2] != shape[2])):
        raise ValueError("q and k must be [tokens, heads, head_dim] with the same tokens and head_dim")
    if k is not None and (k.dtype is not dtype or k.get_device() != device):
        raise ValueError("q and k must have the same dtype and device")
    tokens, heads, dim = shape
    wide = positions.dtype is torch.int64
    if not ((wide or positions.dtype is torch.int32) and positions.get_device() == device and positions.shape == (tokens,)
            and positions.is_contiguous()):
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor [{tokens}] on cuda:{device}")
    double = frequencies.dtype is torch.float64
    if not ((double or frequencies.dtype is torch.float32) and frequencies.get_device() == device and frequencies.dim() == 1
            and frequencies.is_contiguous()):
        raise ValueError(f"frequencies must be a contiguous float64 or float32 tensor on cuda:{device}")
    part = 2 * frequencies.shape[0]
    if not 2 <= part <= dim:
        raise ValueError(f"frequencies must be 1 to {dim // 2}, half of the elements that turn, got {part // 2}")
    if inplace:
        for x in (q, k):
            if x is not None and (x.stride(2) != 1 or not _apart(x)):
                raise ValueError("a tensor that is turned in place has a contiguous last dimension and no element twice")
        if k is not None and q.data_ptr() == k.data_ptr() and q.numel() and k.numel():
            raise ValueError("q and k must not be the same memory")
        a, b = q, k
    else:  # whatever is copied first lives until the launch: its memory must not become an output's
        if q.stride(2) != 1:
            q = q.contiguous()
        a, b = torch.empty_like(q), None
        if k is not None:
            if k.stride(2) != 1:
                k = k.contiguous()
            b = torch.empty_like(k)
    i0, i1, _ = q.stride()
    o0, o1, _ = a.stride()
    side = _ebx.RotarySide(q.data_ptr(), a.data_ptr(), i0, i1, o0, o1, heads, 0)
    other = None
    if k is not None:
        i0, i1, _ = k.stride()
        o0, o1, _ = b.stride()
        other = ctypes.byref(_ebx.RotarySide(k.data_ptr(), b.data_ptr(), i0, i1, o0, o1, k.shape[1], 0))
    st = _ebx.load().ebx_rotate(
        ctypes.byref(side), other, dim, part, _DTYPES[dtype], positions.data_ptr(), 64 if wide else 32,
        frequencies.data_ptr(), 64 if double else 32, tokens, interleaved, scale, device, _stream(device))
    if st:
        _ebx.check(st)
    if inplace:  # a backward pass that saved them must know
        torch.autograd.graph.increment_version(q if k is None else (q, k))
    return a, b


__all__ = ["SCALINGS", "frequencies", "rotate"]
