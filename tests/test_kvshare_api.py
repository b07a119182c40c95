"""What requests that share cache blocks refuse, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mlbricks_b200 import _ebx, kvshare


def test_tensors_on_the_host_are_refused():
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kvshare.fork(i, i.view(1, 1), i, i, torch.zeros(2, dtype=torch.int64), i, block_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        kvshare.compact(i, i.view(1, 1), i, block_size=16)


def test_argument_errors_without_gpu():
    lib = _ebx.load()

    def refused(status, words, code=_ebx.EBX_ERR_INVALID):
        assert status == code
        assert words in _ebx.last_error()

    def fork(lengths=4, tables=4, width=1, block=16, shares=8, blocks=1, ring_size=1, requests=1, out_lengths=8, out_tables=8,
             out_shares=4, ring=8, ring_out=16):
        return lib.ebx_kv_fork(lengths, tables, width, block, shares, blocks, 4, ring_size, ring, 4, None, requests, out_lengths,
                               out_tables, out_shares, ring_out, 4, 4, 0, None)

    refused(fork(lengths=None), "null")
    refused(fork(requests=16385), "16384")
    refused(fork(block=17), "block_size")
    refused(fork(width=2**27), "2^31")
    refused(fork(blocks=2**27), "2^31")
    refused(fork(blocks=0), "blocks")
    refused(fork(ring_size=0), "free_size")
    refused(fork(out_lengths=4), "inputs")
    refused(fork(out_tables=4), "inputs")
    refused(fork(out_shares=8), "inputs")
    refused(fork(ring_out=8), "inputs")

    def compact(width=1, blocks=1, out_tables=8, out_shares=4, sources=4):
        return lib.ebx_kv_compact(4, 4, width, 16, 8, blocks, 1, out_tables, out_shares, 4, 8, sources, sources, 0, None)

    refused(compact(width=0), "width")
    refused(compact(out_tables=4), "inputs")
    refused(compact(out_shares=8), "inputs")
    refused(compact(blocks=2, sources=None), "null")
    refused(compact(blocks=524289), "524288")

    def pools(*changes):
        fields = dict(k_codes=16, k_scales=4, v_codes=16, v_scales=4, blocks=8, kv_heads=2, block_size=16, head_dim=64,
                      device=0, reserved=0)
        return (_ebx.KVPool * len(changes))(*(_ebx.KVPool(*{**fields, **c}.values()) for c in changes))

    refused(lib.ebx_kv_copy(pools({}, dict(blocks=9)), 2, 4, 4, None, 1, None), "same sizes")
    refused(lib.ebx_kv_copy(pools(dict(head_dim=65)), 1, 4, 4, None, 1, None), "head_dim")
    refused(lib.ebx_kv_copy(None, 1, 4, 4, None, 1, None), "null")
    refused(lib.ebx_kv_copy(pools({}), 1, None, 4, None, 1, None), "null")
    refused(lib.ebx_kv_copy(pools({}), 1, 4, 4, None, -1, None), "n >= 0")
    assert lib.ebx_kv_copy(None, 0, None, None, None, 5, None) == _ebx.EBX_OK
    assert lib.ebx_kv_copy(pools({}), 1, None, None, None, 0, None) == _ebx.EBX_OK


@pytest.mark.parametrize("args", [(None, 1, None, None, None, 0)])
def test_copy_without_pools(args):
    assert _ebx.load().ebx_kv_copy(ctypes.cast(None, ctypes.POINTER(_ebx.KVPool)), *args[1:], None) == _ebx.EBX_ERR_INVALID


def test_prefix_errors_without_gpu():
    lib = _ebx.load()

    def refused(status, words, code=_ebx.EBX_ERR_INVALID):
        assert status == code
        assert words in _ebx.last_error()

    def prefixes(tables=4, width=1, block=16, blocks=1, requests=1, tokens=1, out=4):
        return lib.ebx_kv_prefixes(tables, width, block, blocks, 4, 4, requests, tokens, out, 0, None)

    refused(prefixes(tables=None), "null")
    refused(prefixes(out=None), "null")
    refused(prefixes(width=0), "width")
    refused(prefixes(block=1), "block_size")
    refused(prefixes(blocks=0), "blocks")
    refused(prefixes(requests=8193), "8192")
    refused(prefixes(tokens=2**31), "tokens")
    assert prefixes(requests=0, tables=None) == _ebx.EBX_OK
    assert lib.ebx_kv_prefixes_ints(3, 5) == 21 and lib.ebx_kv_prefixes_ints(-1, 5) == 0

    def pool(**change):
        fields = dict(k_codes=16, k_scales=4, v_codes=16, v_scales=4, blocks=8, kv_heads=2, block_size=16, head_dim=64,
                      device=0, reserved=0)
        return ctypes.byref(_ebx.KVPool(*{**fields, **change}.values()))

    def attention(p, heads=4, dtype=1, width=1, scale=1.0, q=16, stride=256, tokens=1, requests=1, shared=4, max_new=0):
        return lib.ebx_kv_shared_attention(p, q, stride, 64, heads, dtype, 4, width, 4, 4, shared, requests, tokens, 1, scale,
                                           max_new, 0, 16, None, None, 0, None)

    refused(attention(None), "null")
    refused(attention(pool(head_dim=96)), "head_dim")
    refused(attention(pool(), heads=3), "multiple of kv_heads")
    refused(attention(pool(), dtype=0), "dtype")
    refused(attention(pool(), scale=float("nan")), "scale")
    refused(attention(pool(), q=8), "aligned")
    refused(attention(pool(), stride=12), "multiples of 8")
    refused(attention(pool(), width=2**27), "out of range")
    refused(attention(pool(), requests=8193), "out of range")
    refused(attention(pool(), shared=None), "null")
    refused(attention(pool(), max_new=-1), ">= 0")
    assert attention(pool(), tokens=0) == _ebx.EBX_OK
    assert lib.ebx_kv_shared_attention_workspace_bytes(pool(head_dim=96), 4, 1, 1, 1, 1) == 0
    takes = lib.ebx_kv_takes_prefixes
    assert takes(pool(), 4, 40, 40, 1, 100000) == 1 and takes(pool(), 4, 40, 40, 1, 0) == 1  # much to read, or unknown
    assert takes(pool(), 4, 40, 40, 1, 500) == 0 and takes(pool(), 4, 40, 40, 25, 100000) == 0  # little; many rows each
    assert takes(pool(blocks=1, kv_heads=2**26, block_size=16), 2**26, 8192, 8192, 0, 2**31 - 1) == 0  # many rows each
    assert takes(pool(blocks=1, kv_heads=2**26, block_size=16), 2**26, 8192, 40, 1, 2**31 - 1) == 1  # a size past 64 bits
    assert takes(pool(), 3, 40, 40, 1, 0) == 0 and takes(pool(), 4, 8193, 40, 1, 0) == 0 and takes(None, 4, 1, 1, 1, 0) == 0
