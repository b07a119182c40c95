"""What the 8-bit cache does with numbers on the device that nobody means: counts, rings and lengths out of
range are not followed, and nothing around the tensors changes."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

kv = pytest.importorskip("mlbricks_b200.kvcache")
MOST = 2**31 - 1


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def guarded(rows, width, value=-1):
    """A table [rows, width] of `value` in the middle of a larger tensor, and that tensor."""
    around = torch.full((rows * width + 8192,), 77, dtype=torch.int32, device="cuda")
    table = around[4096:4096 + rows * width].view(rows, width)
    table.fill_(value)
    return table, around


def test_plan_with_more_tokens_than_31_bits_count():
    """The first two want more than a row holds, and with the second the sum passes 2^31 - 1: nobody gets a block,
    and no token of the room belongs to the last two."""
    tables, around = guarded(4, 1)
    before, free = around.clone(), i32(list(range(8)))
    step = kv.plan(i32([0] * 4), i32([MOST, MOST, 1, 1]), tables, free, i64([0, 8]), block_size=16, tokens=64)
    assert torch.equal(around, before) and free.tolist() == list(range(8))
    assert step.lengths.tolist() == [0] * 4 and step.slots.tolist() == [-1] * 64
    starts = step.starts.tolist()
    assert starts[0] == 0 and starts == sorted(starts)
    assert step.ring[:2].tolist() == [0, 8] and step.ring[3] == 2 * MOST + 2


def test_plan_serves_those_ahead_of_a_sum_that_is_too_large():
    tables, around = guarded(4, 2)
    step = kv.plan(i32([0, 5, 0, 0]), i32([3, 0, MOST, 1]), tables, i32([4, 5, 6]), i64([0, 3]), block_size=16, tokens=3)
    assert step.lengths.tolist() == [3, 5, 0, 0] and step.slots.tolist() == [64, 65, 66]
    assert tables.tolist() == [[4, -1], [-1, -1], [-1, -1], [-1, -1]]
    assert step.ring[:2].tolist() == [1, 3] and step.starts[:3].tolist() == [0, 3, 3]


def test_plan_with_room_for_fewer_tokens_than_there_are():
    """The second request's 17 tokens end past the room for 2: it is refused, and so is the third; the first and
    the one that rests are served, and what leaves the ring is in the table."""
    tables, around = guarded(4, 2, value=55)
    step = kv.plan(i32([0, 0, 0, 9]), i32([1, 17, 1, 0]), tables, i32(list(range(8))), i64([0, 8]), block_size=16, tokens=2)
    assert step.lengths.tolist() == [1, 0, 0, 9] and step.starts.tolist() == [0, 1, 2, 2, 2]
    assert step.slots.tolist() == [0, -1] and step.positions.tolist() == [0, 0]
    assert tables.tolist() == [[0, 55], [55, 55], [55, 55], [55, 55]]
    assert step.ring.tolist() == [1, 8, 3, 19]
    assert (around[:4096] == 77).all() and (around[4104:] == 77).all()


def test_plan_of_a_cache_with_room_for_one_token_a_row():
    """A step captured for one token a row is given two in one row: that row waits, nothing of it is overwritten."""
    cache = kv.KVCache(1, blocks=4, kv_heads=1, head_dim=32, requests=2, max_length=64, block_size=16)
    cache.plan([15, 16])
    step = cache.plan(i32([1, 2]), tokens=2)
    assert cache.lengths.tolist() == [16, 16] and step.slots.tolist() == [15, -1]
    assert cache.ring.tolist() == [2, 4, 1, 3]
    assert cache.plan(i32([0, 2]), tokens=2).ring.tolist() == [3, 4, 0, 2] and cache.lengths.tolist() == [16, 18]


def test_plan_with_a_ring_that_claims_more_than_it_holds():
    """Four blocks, a back 100 places on: nobody gets a block twice, in this step or the next."""
    tables, free = i32([[-1] * 8, [-1] * 8]), i32([0, 1, 2, 3])
    step = kv.plan(i32([0, 0]), i32([128, 0]), tables, free, i64([0, 100]), block_size=16, tokens=128)
    assert step.lengths.tolist() == [0, 0] and step.ring.tolist() == [0, 4, 8, 128]
    assert step.slots.tolist() == [-1] * 128 and (tables == -1).all()
    step = kv.plan(i32([0, 0]), i32([40, 10]), tables, free, i64([1, 100]), block_size=16, tokens=50)
    assert step.lengths.tolist() == [40, 10] and step.ring.tolist() == [5, 5, 0, 50]
    assert tables[:, :4].tolist() == [[1, 2, 3, -1], [0, -1, -1, -1]]
    step = kv.plan(step.lengths, i32([16, 16]), tables, free, step.ring, block_size=16, tokens=32)
    assert step.lengths.tolist() == [40, 10] and step.ring.tolist() == [5, 5, 2, 32]


def test_plan_with_counters_near_their_end():
    """A front and a back at 2^63 - 1, an odd size: the released blocks go to places of the ring."""
    around = torch.full((4096 * 2 + 3,), 77, dtype=torch.int32, device="cuda")
    free = around[4096:4099]
    step = kv.plan(i32([32]), i32([-1]), i32([[8, 9]]), free, i64([2**63 - 1, 2**63 - 1]), block_size=16, tokens=0)
    assert sorted(free.tolist()) == [8, 9, 77] and (around == 77).sum() == around.numel() - 2
    assert step.lengths.tolist() == [0] and int(step.ring[1] - step.ring[0]) == 2


def test_plan_does_not_release_more_than_the_ring_has_places_for():
    free = i32([7, 8, 9])
    step = kv.plan(i32([16, 32]), i32([-1, -1]), i32([[1, 2], [3, 4]]), free, i64([2, 4]), block_size=16, tokens=0)
    assert free.tolist() == [7, 1, 9] and step.ring.tolist() == [2, 5, 0, 0]


def test_plan_keeps_positions_within_31_bits():
    """A length that no table holds: the refused tokens' positions end at 2^31 - 1."""
    step = kv.plan(i32([MOST - 2]), i32([5]), i32([[1]]), i32([2]), i64([0, 1]), block_size=16, tokens=5)
    assert step.positions.tolist() == [MOST - 2, MOST - 1, MOST, MOST, MOST] and step.slots.tolist() == [-1] * 5
    assert step.lengths.tolist() == [MOST - 2]


def test_plan_counts_missing_blocks_past_31_bits():
    """Twenty requests that lack 2^27 blocks each."""
    step = kv.plan(i32([0] * 20), i32([MOST] * 20), i32([[-1]] * 20), i32([0]), i64([0, 1]), block_size=16, tokens=1)
    assert step.ring.tolist() == [0, 1, 20 * 2**27, 20 * MOST]
    assert step.lengths.tolist() == [0] * 20 and step.slots.tolist() == [-1]


def test_attention_with_more_key_tiles_than_31_bits_count():
    """A prompt of 540 thousand tokens in tiles of 8 rows (what a wrong `max_new` leads to): 2.3e9 tiles of 64 keys.

    Tolerance: a weight is rounded to 11 bits (2^-11 of it) and the products' sums to 24 bits, over some 2^13 key
    tiles 2^-11 of their sizes at most; the output's own rounding is 2^-11 of it."""
    n, heads, dim, block = 540_000, 8, 128, 128
    blocks = -(-n // block)
    pool = kv.KVPool(*(t for _ in "kv" for t in (
        torch.randint(-127, 128, (blocks, 1, block, dim), dtype=torch.int8, device="cuda"),
        0.02 * torch.exp(torch.randn(blocks, 1, device="cuda")))))
    table = torch.randperm(blocks, device="cuda").int().view(1, -1)
    q = torch.randn(n, heads, dim, device="cuda", dtype=torch.float16)
    out = torch.full_like(q, 77.0)
    kv.attention(q, pool, table, i32([n]), i32([0, n]), max_new=1, out=out)
    ids = table[0].long()
    k, v = (c[ids].double().mul_(s[ids].double()[..., None, None]).view(-1, dim)[:n]
            for c, s in ((pool.k_codes, pool.k_scales), (pool.v_codes, pool.v_scales)))
    for t in (0, 1, 1000, n // 3, n // 2 + 7, n - 2, n - 1):
        w = torch.softmax(q[t].double() @ k[:t + 1].T / dim**0.5, 1)
        want, size = w @ v[:t + 1], w @ v[:t + 1].abs()
        assert ((out[t].double() - want).abs() <= 2.0**-10 * size + 2.0**-11 * want.abs() + 2.0**-24).all(), t


def test_nobody_overtakes_a_request_that_finds_too_few_blocks():
    """The first lacks 63 blocks of 3; the second needs one and waits, the third needs none and goes on."""
    tables = i32([[5] + [-1] * 63, [6, -1] + [-1] * 62, [7] + [-1] * 63])
    step = kv.plan(i32([16, 16, 3]), i32([1000, 1, 2]), tables, i32([1, 2, 3, 0]), i64([0, 3]), block_size=16, tokens=1003)
    assert step.lengths.tolist() == [16, 16, 5] and step.ring.tolist() == [0, 3, 64, 1003]
    assert step.starts.tolist() == [0, 1000, 1001, 1003]
    assert (step.slots[:1001] == -1).all() and step.slots[1001:].tolist() == [7 * 16 + 3, 7 * 16 + 4]


@pytest.mark.parametrize("new", [1, 60])
def test_a_refused_request_sees_nothing_from_its_length_on(new):
    cache = kv.KVCache(1, blocks=6, kv_heads=1, head_dim=32, requests=2, max_length=96, block_size=16)
    x = torch.randn(42, 1, 32, device="cuda", dtype=torch.float16)
    cache.plan([32, 10])
    cache.append(0, x, x)
    held = cache.lengths.clone()
    step = cache.plan([80, new])  # the first does not fit its row; the second may find its blocks
    fits = new == 1
    assert cache.lengths.tolist() == [32, 10 + new if fits else 10]
    q = torch.randn(80 + new, 2, 32, device="cuda", dtype=torch.float16)
    refused = step.lengths == held
    out, lse = cache.attention(0, q, first=torch.where(refused, step.lengths, 0).int(), return_lse=True)
    gone = step.slots < 0
    assert gone.sum() == (80 if fits else 80 + new)
    assert not out[gone].any() and (lse[gone] == -torch.inf).all() and lse[~gone].isfinite().all()
