"""Numbers of requests at which a kernel's dynamic shared memory nears 48 KB, of which its static shared memory
takes a part: every one of them is launched, each range in a process in which no larger call came before."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PREFIXES = """
import torch
from mlbricks_b200 import kvshare


def found(n):  # all rows begin with the same full block
    i32 = dict(dtype=torch.int32, device="cuda")
    tables = torch.stack([torch.zeros(n, **i32), torch.arange(1, n + 1, **i32)], 1).contiguous()
    starts = torch.arange(n + 1, **i32)
    return kvshare.prefixes(tables, torch.full((n,), 20, **i32), starts, block_size=16, blocks=n + 1, tokens=n)


sizes = range({low}, {high})
first = [found(n) for n in sizes]  # the smaller ones ahead of the larger
found(8192)
for n, one in zip(sizes, first):
    again = found(n)
    assert torch.equal(one.data, again.data), n
    assert (one.data[-1 - n:-1] == 2).all() and int(one.data[-1]) == n, n
"""

PLAN = """
import torch
from mlbricks_b200 import kvcache

for n in range({low}, {high}):
    i32 = dict(dtype=torch.int32, device="cuda")
    tables = torch.full((n, 1), -1, **i32)
    step = kvcache.plan(torch.zeros(n, **i32), torch.ones(n, **i32), tables, torch.arange(n, **i32),
                        torch.tensor([0, n, 0, 0], device="cuda"), block_size=16, tokens=n)
    assert torch.equal(tables[:, 0], torch.arange(n, **i32)), n
    assert (step.lengths == 1).all() and step.ring.tolist() == [n, n, 0, n], n
    assert torch.equal(step.starts, torch.arange(n + 1, **i32)) and torch.equal(step.slots, 16 * torch.arange(n, device="cuda")), n
"""


# 2048 sorted places of 8 bytes and 20 bytes a request reach 48 KB behind 1638 requests, 12 bytes a request at 4096
@pytest.mark.parametrize("program, low, high", [(PREFIXES, 1600, 1642), (PLAN, 4060, 4099)], ids=["prefixes", "plan"])
def test_requests_near_48_kb(cuda_ok, program, low, high):
    done = subprocess.run([sys.executable, "-c", program.format(low=low, high=high)], cwd=Path(__file__).resolve().parents[1],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
