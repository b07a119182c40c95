"""The cache's public surface and the argument checks that need no GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mlbricks_b200 import _ebx, kvcache


def test_public_names():
    assert set(kvcache.__all__) == {"BLOCK_SIZES", "HEAD_DIMS", "KVCache", "KVPlan", "KVPool", "append", "attention",
                                    "materialize", "plan"}


def test_tensors_on_the_host_are_refused():
    codes, scales = torch.zeros(2, 1, 16, 32, dtype=torch.int8), torch.zeros(2, 1)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.KVPool(codes, scales, codes, scales)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.plan(i, i, i.view(1, 1), i, torch.zeros(2, dtype=torch.int64), block_size=16, tokens=0)


def test_argument_errors_without_gpu():
    lib = _ebx.load()

    def pool(**change):
        fields = dict(k_codes=16, k_scales=4, v_codes=16, v_scales=4, blocks=8, kv_heads=2, block_size=16, head_dim=64,
                      device=0, reserved=0)
        return ctypes.byref(_ebx.KVPool(*{**fields, **change}.values()))

    def attention(p, heads=4, dtype=1, width=1, window=0, causal=1, scale=1.0, q=16, stride=256, tokens=1):
        return lib.ebx_kv_attention(p, q, stride, 64, heads, dtype, 4, width, 4, 4, None, 1, tokens, causal, window,
                                    scale, 0, 0, 16, None, None, 0, None)

    def refused(status, words):
        assert status == _ebx.EBX_ERR_INVALID
        assert words in _ebx.last_error()

    refused(attention(None), "null")
    refused(attention(pool(k_codes=None)), "null")
    refused(attention(pool(block_size=24)), "block_size")
    refused(attention(pool(head_dim=96)), "head_dim")
    refused(attention(pool(blocks=2**27)), "2^31")
    refused(attention(pool(k_codes=8)), "aligned")
    refused(attention(pool(), heads=3), "multiple of kv_heads")
    refused(attention(pool(), dtype=0), "dtype")
    refused(attention(pool(), window=-1), "window")
    refused(attention(pool(), window=3, causal=0), "window")
    refused(attention(pool(), scale=float("nan")), "scale")
    refused(attention(pool(), q=8), "aligned")
    refused(attention(pool(), stride=12), "multiples of 8")
    refused(attention(pool(), width=2**27), "out of range")
    assert attention(pool(), tokens=0) == _ebx.EBX_OK
    refused(lib.ebx_kv_append(pool(), 16, 128, 64, 16, 128, 64, 8, 1, 0, None), "dtype")
    refused(lib.ebx_kv_append(pool(), 16, 128, 64, 16, 128, 4, 8, 1, 1, None), "multiples of 8")
    refused(lib.ebx_kv_materialize(pool(), 4, 1, 4, None, 1, 1, 3, 16, 16, None), "dtype")
    refused(lib.ebx_kv_plan(4, 4, 16385, 4, 1, 16, 4, 1, 8, 16, 8, 4, 8, 4, 1, 0, None), "16384")
    refused(lib.ebx_kv_plan(4, 4, 1, 4, 1, 17, 4, 1, 8, 16, 8, 4, 8, 4, 1, 0, None), "block_size")
    refused(lib.ebx_kv_plan(4, 4, 1, 4, 1, 16, 4, 1, 8, 8, 16, 4, 8, 4, 1, 0, None), "ring_out")
    assert lib.ebx_kv_attention_workspace_bytes(pool(head_dim=96), 4, 1, 1, 1) == 0
