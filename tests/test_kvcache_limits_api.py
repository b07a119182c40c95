"""Sizes that the cache's C entries refuse before anything reaches a GPU."""
from __future__ import annotations

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
