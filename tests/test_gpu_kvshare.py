"""Forking, freeing, compacting and copying cache blocks against plain lists: equal to the last number."""
from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

kv = pytest.importorskip("mlbricks_b200.kvcache")
share = pytest.importorskip("mlbricks_b200.kvshare")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def blocks_of(n, b):
    return -(-n // b)


class Rows:
    """Rows of a table as lists of blocks, their holders, and the ring."""

    def __init__(self, lengths, rows, holders, ring, block):
        self.lengths, self.rows, self.holders, self.ring, self.block = lengths, rows, holders, ring, block

    def fork(self, parents, keep=None):
        """The copies (source, target), the blocks that were missing, and the places of the ring taken."""
        b, n = self.block, len(self.lengths)
        old_rows, old_lengths = [list(r) for r in self.rows], list(self.lengths)
        new = []
        for r, p in enumerate(parents):
            have = old_lengths[p] if 0 <= p < n else 0
            new.append(min(have, max(keep[r], 0)) if keep else have)
        changed = [parents[r] != r or new[r] != old_lengths[r] for r in range(n)]
        for r in range(n):
            if changed[r]:
                for x in old_rows[r]:
                    self.holders[x] -= 1
                for x in old_rows[parents[r]][:new[r] // b] if new[r] else []:
                    self.holders[x] += 1
        wanted = {}  # begun block -> rows that want it, the parent itself first
        for r in sorted(range(n), key=lambda r: (parents[r] != r, r)):
            if changed[r] and new[r] % b:
                x = old_rows[parents[r]][new[r] // b]
                if self.holders[x] == 0:
                    wanted.setdefault(x, r)
        copies, missing = [], 0
        for r in range(n):
            if not changed[r]:
                continue
            row = old_rows[parents[r]][:blocks_of(new[r], b)] if new[r] else []
            if new[r] % b:
                x = row[-1]
                if wanted.get(x) == r:
                    self.holders[x] += 1
                elif self.ring:
                    row = row[:-1] + [self.ring.pop(0)]
                    self.holders[row[-1]] += 1
                    copies.append((x, row[-1]))
                else:
                    for y in row[:-1]:
                        self.holders[y] -= 1
                    row, new[r] = [], 0
                    missing += 1
            self.rows[r], self.lengths[r] = row, new[r]
        held = {x for row in old_rows for x in row}
        self.ring += sorted(x for x in held if self.holders[x] == 0)
        return copies, missing

    def tensors(self, width, front=0, extra=0):
        """lengths, tables, shares, free, ring as the operators take them."""
        total = len(self.holders)
        size = total + extra
        free = torch.full((size,), -7, dtype=torch.int32)
        for j, x in enumerate(self.ring):
            free[(front + j) % size] = x
        tables = torch.full((len(self.rows), width), 12345678, dtype=torch.int32)  # not to be followed
        for i, row in enumerate(self.rows):
            tables[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        shares = [max(h - 1, 0) for h in self.holders]
        return i32(self.lengths), tables.cuda(), i32(shares), free.cuda(), i64([front, front + len(self.ring), 5, 5])


def ring_list(free, ring):
    front, back = int(ring[0]), int(ring[1])
    return [int(free[j % free.numel()]) for j in range(front, back)]


def random_rows(rng, requests, block, most, spare):
    """Rows some of which share the full blocks of another's beginning."""
    rows, lengths, count = [], [], 0
    for i in range(requests):
        n = rng.choice([0, rng.randrange(most + 1), rng.randrange(most + 1), block * rng.randrange(most // block + 1)])
        row = []
        if rows and rng.random() < 0.5:
            other = rng.randrange(len(rows))
            row = rows[other][:min(n // block, rng.randrange(lengths[other] // block + 1))]
        more = blocks_of(n, block) - len(row)
        rows.append(row + list(range(count, count + more)))
        lengths.append(n)
        count += more
    total = max(count + spare, 1)
    names = list(range(total))
    rng.shuffle(names)
    rows = [[names[x] for x in row] for row in rows]
    holders = [0] * total
    for row in rows:
        for x in row:
            holders[x] += 1
    ring = [x for x in range(total) if holders[x] == 0]
    rng.shuffle(ring)
    return Rows(lengths, rows, holders, ring, block)


def check_fork(rows, parents, keep=None, front=0, extra=0, width=None):
    width = width or max([len(r) for r in rows.rows] + [1])
    lengths, tables, shares, free, ring = rows.tensors(width, front, extra)
    before = [t.clone() for t in (lengths, tables, shares, ring)]
    took = len(rows.ring)
    got = share.fork(lengths, tables, shares, free, ring, i32(parents), block_size=rows.block,
                     keep=None if keep is None else i32(keep))
    assert all(torch.equal(x, y) for x, y in zip(before, (lengths, tables, shares, ring)))
    copies, missing = rows.fork(parents, keep)
    assert got.lengths.tolist() == rows.lengths
    want = [row + [-1] * (width - len(row)) for row in rows.rows]
    assert got.tables.tolist() == want
    assert got.shares.tolist() == [max(h - 1, 0) for h in rows.holders]
    assert got.ring[2:].tolist() == [missing, len(copies)]
    assert int(got.ring[0]) == front + len(copies)
    assert ring_list(free, got.ring) == rows.ring, (took, copies)
    n = len(parents)
    assert got.moves.sources.tolist() == [s for s, _ in copies] + [-1] * (n - len(copies))
    assert got.moves.targets.tolist() == [t for _, t in copies] + [-1] * (n - len(copies))
    assert int(got.moves.count) == len(copies)
    return got


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_fork_random(block):
    rng = random.Random(block)
    for requests, most in ((1, 5 * block), (2, 3 * block), (7, 9 * block), (40, 4 * block), (40, 70 * block), (300, 3 * block)):
        for _ in range(3):
            rows = random_rows(rng, requests, block, most, rng.choice([0, 3, requests]))
            for kind in range(3):  # one after the other on the same rows
                parents = [rng.choice([i, i, -1, rng.randrange(requests), rng.randrange(requests)]) for i in range(requests)]
                keep = None if kind == 0 else [rng.choice([2**31 - 1, -1, n, n - 1, rng.randrange(most + 1)]) for n in rows.lengths]
                front = rng.choice([0, 3, 2**40 + 17])
                check_fork(rows, parents, keep, front=front, extra=rng.choice([0, 5]))


def test_fork_nothing_changes():
    rows = random_rows(random.Random(5), 9, 16, 100, 4)
    got = check_fork(rows, list(range(9)))
    assert got.ring[2:].tolist() == [0, 0]


def test_fork_of_everyone_and_free_of_all():
    """All rows from one; then all freed at once: each block to the ring once."""
    n = 50
    rows = Rows([100] + [0] * (n - 1), [list(range(7))] + [[] for _ in range(n - 1)], [1] * 7 + [0] * n, list(range(7, 7 + n)), 16)
    got = check_fork(rows, [0] * n)
    assert int(got.moves.count) == n - 1 and got.shares[:6].tolist() == [n - 1] * 6
    got = check_fork(rows, [-1] * n, front=3)
    assert ring_list_len(got) == 7 + n


def ring_list_len(got):
    return int(got.ring[1] - got.ring[0])


def test_fork_without_blocks_left():
    """Rows that find no block hold nothing, and what they took is let go."""
    rows = Rows([40, 0, 0, 0], [[2, 0, 1], [], [], []], [1, 1, 1, 0], [3], 16)
    got = check_fork(rows, [0, 0, 0, 0])
    assert got.lengths.tolist() == [40, 40, 0, 0] and got.ring.tolist()[2:] == [2, 1]
    # the parent's row goes to another, and those that are refused were the only holders
    rows = Rows([40, 33], [[2, 0, 1], [4, 3, 5]], [1] * 6, [], 16)
    got = check_fork(rows, [-1, -1])
    rows = Rows([40, 0, 0], [[2, 0, 1], [], []], [1, 1, 1], [], 16)
    got = check_fork(rows, [-1, 0, 0])  # row 1 keeps the begun block
    assert got.lengths.tolist() == [0, 40, 0]


def test_roll_back_into_a_shared_block():
    """A row rolled back into a block that another holds whole needs a copy; into one that all leave, the first keeps it."""
    rows = Rows([48, 50], [[0, 1, 2], [0, 1, 2, 3]], [2, 2, 2, 1, 0, 0], [4, 5], 16)
    got = check_fork(rows, [0, 1], [40, 50])
    assert got.tables.tolist()[0][:3] == [0, 1, 4] and got.shares.tolist() == [1, 1, 0, 0, 0, 0]
    rows = Rows([48, 50], [[0, 1, 2], [0, 1, 2, 3]], [2, 2, 2, 1, 0, 0], [4, 5], 16)
    got = check_fork(rows, [0, 1], [40, 41])
    assert got.tables.tolist()[0][:3] == [0, 1, 2] and got.tables.tolist()[1][:3] == [0, 1, 4]


def test_fork_large():
    rng = random.Random(1)
    rows = random_rows(rng, 2500, 16, 200, 1500)
    check_fork(rows, [rng.randrange(-1, 2500) for _ in range(2500)], front=11)
    rows = random_rows(rng, 3, 16, 300000, 9)
    check_fork(rows, [2, 0, 0])


def test_numbers_out_of_range_are_not_followed():
    """Lengths past the row, blocks that are none, parents that are none: nothing outside is touched."""
    lengths, tables = i32([2**31 - 1, -5, 33, 20]), i32([[0, 99, -3], [1, 1, 1], [2, 3, 2**31 - 1], [-1, 50, 4]])
    shares, free, ring = i32([0] * 6), i32([5, 0, 0, 0, 0, 0]), i64([0, 1, 0, 0])
    got = share.fork(lengths, tables, shares, free, ring, i32([0, 7, 1, 3]), block_size=16)
    # row 0 is cut to its width and stays, row 1's parent is none, row 2 takes row 1's nothing, row 3 stays
    assert got.lengths.tolist() == [2**31 - 1, 0, 0, 20] or got.lengths.tolist() == [48, 0, 0, 20]
    assert got.tables.tolist()[3] == [-1, 50, -1] and got.ring.tolist() == [0, 3, 0, 0]
    got = share.fork(lengths, tables, shares, free, ring, i32([2, 2, 2, 2]), block_size=16)
    assert got.lengths.tolist() == [33] * 4  # the begun entry is no block: it is kept, and nothing is copied
    assert got.ring.tolist()[2:] == [0, 0]
    # a ring that claims more than it holds, and counters near 2^63
    for claimed in ([0, 100], [2**63 - 50, 2**63 - 44], [-9, 2]):
        got = share.fork(i32([20, 0]), i32([[0, 1], [-1, -1]]), i32([0] * 4), i32([2, 3, 2, 3]), i64(claimed), i32([0, 0]), block_size=16)
        assert got.lengths.tolist() == [20, 20] and int(got.ring[3]) == 1


@pytest.mark.parametrize("block", [16, 128])
def test_compact(block):
    rng = random.Random(block + 1)
    for requests, most, spare in ((1, 3 * block, 0), (1, 0, 1), (5, 4 * block, 0), (6, 9 * block, 100), (200, 5 * block, 700), (3, 2000 * block, 900), (2, 7 * block, 200000)):
        rows = random_rows(rng, requests, block, most, spare)
        width = max([len(r) for r in rows.rows] + [1]) + 2
        lengths, tables, shares, _, _ = rows.tensors(width)
        total = len(rows.holders)
        if total == 0:
            continue
        got = share.compact(lengths, tables, shares, block_size=block)
        held = sorted({x for r in rows.rows for x in r})
        count = len(held)
        high = [x for x in held if x >= count]
        low = [x for x in range(count) if x not in set(held)]
        to = {**{x: x for x in held}, **dict(zip(high, low))}
        assert len(high) == len(low)
        assert got.tables.tolist() == [[to[x] for x in r] + [-1] * (width - len(r)) for r in rows.rows]
        want = [0] * total
        for x in held:
            want[to[x]] = rows.holders[x] - 1
        assert got.shares.tolist() == want
        assert got.free.tolist() == list(range(count, total)) + [-1] * count
        assert got.ring.tolist() == [0, total - count, 0, len(high)]
        pad = [-1] * (total // 2 - len(high))
        assert got.moves.sources.tolist() == high + pad and got.moves.targets.tolist() == low + pad


@pytest.mark.parametrize("heads, block, dim, layers", [(1, 16, 32, 1), (3, 32, 64, 5), (8, 64, 128, 2), (5, 128, 128, 3), (1, 32, 32, 70)])
def test_copy(heads, block, dim, layers):
    blocks = 23
    pools, before = [], []
    for _ in range(layers):
        codes = [torch.randint(-127, 128, (blocks, heads, block, dim), dtype=torch.int8, device="cuda") for _ in "kv"]
        scales = [torch.rand(blocks, heads, device="cuda") for _ in "kv"]
        pools.append(kv.KVPool(codes[0], scales[0], codes[1], scales[1]))
        before.append([t.clone() for t in (codes[0], scales[0], codes[1], scales[1])])
    sources, targets = i32([0, 22, 3, 3, -1, 5, 23, 9]), i32([1, 7, 4, 21, 2, -1, 8, 10])
    for count, real in ((None, [0, 1, 2, 3, 7]), (i64([3]), [0, 1, 2]), (i64([0]), []), (i64([99]), [0, 1, 2, 3, 7]), (i64([-4]), [])):
        share.copy(pools, share.KVMoves(sources, targets, count))
        for pool, old in zip(pools, before):
            for t, o in zip((pool.k_codes, pool.k_scales, pool.v_codes, pool.v_scales), old):
                o[targets[real].long()] = o[sources[real].long()]
                assert torch.equal(t, o)
                t.copy_(o)


def test_other_stream_and_graph():
    """A captured fork and copy, replayed, goes by what the tensors then hold."""
    rng = random.Random(2)
    rows = random_rows(rng, 12, 32, 300, 20)
    width = max(len(r) for r in rows.rows) + 1
    lengths, tables, shares, free, ring = rows.tensors(width)
    pool = kv.KVPool.empty(len(rows.holders), 2, 32, 64)
    parents = i32([0] * 12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        share.copy([pool], share.fork(lengths, tables, shares, free.clone(), ring, parents, block_size=32).moves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = share.fork(lengths, tables, shares, free, ring, parents, block_size=32)
        share.copy([pool], held.moves)
    pool.k_codes.random_(-127, 128)
    codes = pool.k_codes.clone()
    choice = [rng.randrange(12) for _ in range(12)]
    parents.copy_(i32(choice))
    graph.replay()
    copies, _ = rows.fork(choice)
    assert held.lengths.tolist() == rows.lengths and ring_list(free, held.ring) == rows.ring
    for s, t in copies:
        codes[t] = codes[s]
    assert torch.equal(pool.k_codes, codes)


def test_refusals():
    lengths, tables, shares, free, ring = i32([1]), i32([[0, 1]]), i32([0, 0]), i32([0, 1]), i64([0, 1])
    parents = i32([0])
    for change, words in [(dict(lengths=lengths.long()), "lengths"), (dict(tables=tables.cpu()), "tables"),
                          (dict(shares=shares.float()), "shares"), (dict(ring=ring.int()), "ring"),
                          (dict(parents=i32([0, 0])), "parents"), (dict(keep=i32([0, 0])), "parents and keep"),
                          (dict(block_size=8), "block_size"), (dict(tables=i32([[0], [1]])), "a row for each"),
                          (dict(free=free.long()), "free"), (dict(shares=shares[:0]), "shares"),
                          (dict(tables=i32([[0, 1, 2, 3]])[:, ::2]), "tables")]:
        args = {**dict(lengths=lengths, tables=tables, shares=shares, free=free, ring=ring, parents=parents, block_size=16), **change}
        with pytest.raises(ValueError, match=words):
            share.fork(**args)
    none = share.fork(lengths[:0], tables[:0], shares, free, ring, parents[:0], block_size=16)
    assert none.lengths.numel() == 0 and none.ring.tolist() == [0, 1, 0, 0]
    with pytest.raises(ValueError, match="16384"):
        share.fork(i32([0]).repeat(16385), i32([[0]]).repeat(16385, 1), shares, free, ring, i32([0]).repeat(16385), block_size=16)
    a, b = kv.KVPool.empty(2, 1, 16, 32), kv.KVPool.empty(3, 1, 16, 32)
    moves = share.KVMoves(i32([0]), i32([1]), None)
    with pytest.raises(ValueError, match="same sizes"):
        share.copy([a, b], moves)
    with pytest.raises(ValueError, match="as many"):
        share.copy([a], share.KVMoves(i32([0]), i32([1, 0]), None))
    with pytest.raises(ValueError, match="sources"):
        share.copy([a], share.KVMoves(torch.zeros(1, dtype=torch.int32), i32([1]), None))
    share.copy([], moves)


def test_offsets_past_32_bits():
    """A pool of 8.6 GB of codes a side: blocks at both of its ends."""
    blocks = 131072
    pool = kv.KVPool(*(t for _ in "kv" for t in (torch.empty(blocks, 8, 64, 128, dtype=torch.int8, device="cuda"),
                                                 torch.empty(blocks, 8, device="cuda"))))
    for t in (pool.k_codes, pool.v_codes):
        t[0].random_(-127, 128), t[-1].random_(-127, 128)
    for t in (pool.k_scales, pool.v_scales):
        t[0].uniform_(), t[-1].uniform_()
    moves = share.KVMoves(i32([blocks - 1, 0]), i32([1, blocks - 2]), None)
    share.copy([pool], moves)
    for t in (pool.k_codes, pool.k_scales, pool.v_codes, pool.v_scales):
        assert torch.equal(t[1], t[-1]) and torch.equal(t[-2], t[0])
    got = share.compact(i32([200, 64]), i32([[blocks - 1, 5, blocks - 2, 0], [77777, -1, -1, -1]]), i32([0]).repeat(blocks), block_size=64)
    assert got.tables.tolist() == [[4, 1, 3, 0], [2, -1, -1, -1]]  # 5, 77777 and the last two, in that order, to 1 .. 4
    assert got.ring.tolist()[1] == blocks - 5
