"""The example that serves a compressed decoder over the cache, and KVCache's own bookkeeping.

Tolerance, from the arithmetic: a code is off by at most half a step, on average step / sqrt(12);
with the largest of a block's 1024 normal values near 3.3 of their size, that is 3.3 / 127 / sqrt(12)
= 0.75 % of a value.  Keys and values each bring that into an attention output, which the residual
stream and three layers add up in squares: 0.75 % * sqrt(2 * 3) = 1.8 %; 5 % leaves room for a layer
that enlarges it."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def test_serving_a_compressed_decoder(cuda_ok):
    import kv_serving

    result = kv_serving.serve(steps=24)
    held = [5 + 24, 200 + 12, 64 + 24, 333 + 24]
    assert result["lengths"] == held
    assert result["texts"] == [n + 1 for n in held]
    assert result["missing"] == 0
    assert result["free"] == 40 - sum(-(-n // 32) for n in held)
    assert max(result["errors"]) < 0.05


def test_blocks_run_out_and_come_back(cuda_ok):
    from mlbricks_b200.kvcache import KVCache

    cache = KVCache(1, blocks=4, kv_heads=1, head_dim=32, requests=3, max_length=64, block_size=16)
    assert cache.plan([20, 17, 1]).ring.tolist() == [4, 4, 1, 38]  # the third finds none left
    assert cache.lengths.tolist() == [20, 17, 0]
    assert cache.step.slots[-1] == -1
    assert cache.plan([-1, 0, 0]).ring.tolist() == [4, 6, 0, 0]
    assert cache.plan([0, 15, 1]).ring.tolist() == [5, 6, 0, 16]
    assert cache.lengths.tolist() == [0, 32, 1]
    assert cache.plan([65, 0, 0]).ring.tolist() == [5, 6, 5, 65]   # longer than a row of the table
    with pytest.raises(ValueError, match="tokens"):
        cache.plan(torch.ones(3, dtype=torch.int32, device="cuda"))
    fresh = KVCache(1, blocks=4, kv_heads=1, head_dim=32, requests=3, max_length=64, block_size=16)
    with pytest.raises(RuntimeError, match="plan"):
        fresh.attention(0, torch.zeros(1, 1, 32, device="cuda", dtype=torch.float16))
