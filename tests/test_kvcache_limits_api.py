"""Sizes that the cache's C entries refuse before anything reaches a GPU."""
from __future__ import annotations

import ctypes

import pytest

from mlbricks_b200 import _ebx


def refused(status, words):
    assert status == _ebx.EBX_ERR_INVALID
    assert words in _ebx.last_error()


@pytest.mark.parametrize("width,block", [(2**24, 128), (2**27, 16), (2**31 - 1, 64)])
def test_plan_refuses_rows_that_hold_more_tokens_than_a_length_counts(width, block):
    """A request in such a row could pass 2^31 - 1 tokens: its positions would turn negative, and its table
    entries lie ahead of the table."""
    lib = _ebx.load()
    refused(lib.ebx_kv_plan(4, 4, 1, 4, width, block, 4, 1, 8, 16, 8, 4, 8, 4, 1, 0, None), "2^31")


def pool(**change):
    fields = dict(k_codes=16, k_scales=4, v_codes=16, v_scales=4, blocks=8, kv_heads=2, block_size=16, head_dim=64,
                  device=0, reserved=0)
    return ctypes.byref(_ebx.KVPool(*{**fields, **change}.values()))


@pytest.mark.parametrize("tokens", [2**31, 2**62, 2**63 - 1])
def test_attention_refuses_more_rows_than_it_counts(tokens):
    """2^62 tokens of four heads a key/value head are 2^64 rows, which 64 bits show as none."""
    lib = _ebx.load()
    refused(lib.ebx_kv_attention(pool(), 16, 256, 64, 8, 1, 4, 1, 4, 4, None, 1, tokens, 1, 0, 1.0, 0, 0, 16, None, None,
                                 0, None), "out of range")
    assert lib.ebx_kv_attention_workspace_bytes(pool(), 8, tokens, 0, 0) == 0


@pytest.mark.parametrize("kv_heads,head_dim", [(2**24, 128), (2**27 - 1, 32)])
def test_materialize_refuses_tokens_wider_than_it_counts(kv_heads, head_dim):
    """The elements of a CTA's 16 tokens, 16 to a thread, would pass 31 bits, and nothing would be written."""
    lib = _ebx.load()
    wide = pool(blocks=1, kv_heads=kv_heads, head_dim=head_dim)
    refused(lib.ebx_kv_materialize(wide, 4, 1, 4, None, 1, 1, 1, 16, 16, None), "2^30")


def test_attention_without_requests_has_nothing_to_do():
    """Rows of no request are left as they are: that is no error."""
    lib = _ebx.load()
    assert lib.ebx_kv_attention(pool(), 16, 256, 64, 4, 1, None, 1, None, 4, None, 0, 5, 1, 0, 1.0, 0, 0, 16, None, None,
                                0, None) == _ebx.EBX_OK
