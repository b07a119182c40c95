"""Attention over shared prefixes against the formula in 64 bits.

Tolerances: those of tests/test_gpu_kvcache.py, whose derivation holds for the results over the prefix and over the rest
alike (weights of 11 bits, sums in fp32); joining the two multiplies each by a power of two of which the exponent is
off by 2^-22 at most and adds them, some 2^-21 of their sizes, which the factor 2 in 2^-10 |w v| covers.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from test_gpu_kvcache import check_attention, i32, make_pool

pytestmark = pytest.mark.gpu

kv = pytest.importorskip("mlbricks_b200.kvcache")
share = pytest.importorskip("mlbricks_b200.kvshare")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def blocks_of(n, b):
    return -(-n // b)


def make_tables(groups, lengths, prefix, block, spare=2, width=None):
    """Rows of request i with groups[i] >= 0 begin with the prefix[groups[i]] // block blocks of that group; entries that no
    token needs are garbage."""
    common = [p // block for p in prefix]
    count = sum(common) + sum(blocks_of(n, block) for n in lengths) + spare
    order = torch.randperm(count).tolist()
    at = [sum(common[:g]) for g in range(len(prefix))]
    heads = [order[a:a + c] for a, c in zip(at, common)]
    place = sum(common)
    width = width or max(1, max(blocks_of(n, block) for n in lengths) + 1)
    tables = torch.randint(-(2**31), 2**31 - 1, (len(lengths), width), dtype=torch.int64).int()
    for i, (g, n) in enumerate(zip(groups, lengths)):
        need = blocks_of(n, block)
        row = (heads[g] if g >= 0 else [])[:need]
        more = need - len(row)
        row = row + order[place:place + more]
        place += more
        tables[i, :need] = torch.tensor(row, dtype=torch.int32)
    return tables.cuda(), count


def states(found):
    """Of each token: 0: of no request, 1: of a request by itself, 2: of one in a group."""
    return found.data[-1 - found.tokens:-1]


def run(groups, prefix, lengths, new, *, heads, group, dim, block, dtype=torch.float16, q_size=1.0, grouped=None, tail=0, **kw):
    tables, blocks = make_tables(groups, lengths, prefix, block)
    pool = make_pool(blocks, heads, block, dim)
    tokens = sum(new) + tail
    fused = q_size * torch.randn(tokens, heads * group + 3, dim, device="cuda")
    q = fused.to(dtype)[:, 1:1 + heads * group]
    starts = i32([sum(new[:i]) for i in range(len(new) + 1)])
    found = share.prefixes(tables, i32(lengths), starts, block_size=block, blocks=blocks, tokens=tokens)
    if grouped is not None:
        assert int((states(found) == 2).sum()) == grouped
    out = torch.full((tokens, heads * group, dim), 7.0, dtype=dtype, device="cuda")
    _, lse = share.attention(q, pool, tables, i32(lengths), starts, found, return_lse=True, out=out, **kw)
    kw.pop("max_new", None), kw.pop("max_length", None)
    check_attention(q, pool, tables, lengths, new, out, lse, **kw)
    assert (out[sum(new):] == 7.0).all()  # rows of no request
    return q, pool, tables, starts, found, out, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads, group", [(1, 12), (2, 4), (3, 1), (1, 40)])
def test_one_group(dtype, dim, heads, group):
    """From two members to many, so that either kernel takes the prefix, behind odd lengths."""
    for members, block in ((2, 16), (5, 64), (17, 32), (70, 128)):
        prefix = 3 * block + 5
        lengths = [prefix + 1 + 7 * i % 90 for i in range(members)]
        run([0] * members, [prefix], lengths, [1] * members, heads=heads, group=group, dim=dim, block=block, dtype=dtype,
            grouped=members, max_new=1)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("heads, group, dim", [(2, 4, 128), (1, 12, 32), (4, 1, 64)])
def test_groups_among_others(block, heads, group, dim):
    """Several groups whose members are not neighbours, some requests alone, some without tokens, several tokens each."""
    rng = random.Random(block)
    for most in (1, 4):
        requests = 41
        groups = [rng.choice([-1, 0, 0, 1, 2, 2, 2]) for _ in range(requests)]
        prefix = [5 * block + 3, 2 * block, 900]
        new = [rng.choice([0, 1, most, rng.randint(1, most)]) for _ in range(requests)]
        lengths = [(prefix[g] if g >= 0 else 0) + rng.randrange(200) + n for g, n in zip(groups, new)]
        run(groups, prefix, lengths, new, heads=heads, group=group, dim=dim, block=block, max_new=most, tail=3)
        run(groups, prefix, lengths, new, heads=heads, group=group, dim=dim, block=block, max_new=most, dtype=torch.bfloat16,
            causal=False, scale=0.21)


def test_long_prefixes_are_split():
    for members, prefix in ((4, 40000), (40, 20001)):
        lengths = [prefix + 1 + 50 * i for i in range(members)]
        run([0] * members, [prefix], lengths, [1] * members, heads=2, group=4, dim=128, block=64, max_new=1,
            max_length=max(lengths), grouped=members)


def test_many_groups_and_requests():
    """More requests than the shares count at once, groups of two."""
    requests = 1300
    groups = [i % 650 for i in range(requests)]
    lengths = [34 + i % 20 for i in range(requests)]
    run(groups, [32] * 650, lengths, [1] * requests, heads=1, group=4, dim=32, block=16, max_new=1, grouped=requests)


def test_nobody_shares():
    lengths = [1, 100, 37, 0, 16]
    run([-1] * 5, [], lengths, [1, 1, 2, 0, 1], heads=2, group=4, dim=64, block=16, max_new=2, grouped=0)


def test_requests_that_hold_nothing():
    """New tokens of a request of length 0, or of fewer than it brings, see nothing and get 0."""
    q, pool, tables, starts, found, out, lse = run([0, 0, 0, -1], [40], [60, 61, 45, 0], [1, 1, 1, 2], heads=2, group=4, dim=64,
                                                   block=16, max_new=2, grouped=3)
    assert torch.equal(out[3:5], torch.zeros_like(out[3:5])) and torch.isneginf(lse[3:5]).all()


def test_who_joins():
    """The common length that saves most reading is taken; who has less in common goes alone, and so does a row whose new
    tokens lie in the block."""
    block = 16
    tables = i32([[1, 2, 3, 4, 5, 6], [1, 2, 3, 4, 7, 8], [1, 2, 3, 4, 9, 10], [1, 20, 21, 22, 23, 24], [1, 2, 3, 4, 11, 12], [1, 30, 31, 32, 33, 34]])
    starts = i32(range(7))
    shared = share.prefixes(tables, i32([90] * 6), starts, block_size=block, blocks=40, tokens=6)
    state = states(shared).tolist()
    assert state == [2, 2, 2, 1, 2, 1]  # 3 * 4 blocks rather than 5 * 1
    shared = share.prefixes(tables, i32([90, 90, 90, 90, 64, 16]), starts, block_size=block, blocks=40, tokens=6)
    assert states(shared).tolist() == [2, 2, 2, 1, 2, 1]  # 3 members of 4 blocks or 4 of 3: 8 or 9
    shared = share.prefixes(tables, i32([90, 90, 16, 16, 16, 16]), starts, block_size=block, blocks=40, tokens=6)
    assert states(shared).tolist() == [2, 2, 1, 1, 1, 1]


def test_same_as_without_prefixes():
    """The same formula: both within their tolerances; and with many rows of its own a request goes alone, bit for bit."""
    groups, lengths, new = [0] * 6, [3000 + 11 * i for i in range(6)], [60] * 6
    q, pool, tables, starts, found, out, lse = run(groups, [2900], lengths, new, heads=2, group=4, dim=64, block=32, max_new=60)
    want, want_lse = kv.attention(q, pool, tables, i32(lengths), starts, max_new=60, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert torch.equal(share.attention(q, pool, tables, i32(lengths), starts, found, max_new=60), want)


def test_results_do_not_depend_on_luck():
    args = dict(heads=8, group=4, dim=128, block=64, max_new=1)
    q, pool, tables, starts, found, out, lse = run([0] * 30 + [1] * 9, [5000, 300], [5100] * 30 + [333] * 9, [1] * 39, **args)
    for _ in range(3):
        again, again_lse = share.attention(q, pool, tables, i32([5100] * 30 + [333] * 9), starts, found, max_new=1, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


def test_large_scores_and_values_that_are_not_finite():
    q, pool, tables, starts, found, out, _ = run([0] * 20, [200], [230] * 20, [1] * 20, heads=1, group=4, dim=64, block=32,
                                                 q_size=20.0, max_new=1)
    lengths = i32([230] * 20)
    # a block that only request 3 holds: its rows alone
    pool.v_scales[tables[3, 6].long()] = math.nan
    got = share.attention(q, pool, tables, lengths, starts, found, max_new=1)
    assert torch.isnan(got[3]).all() and torch.equal(got[:3], out[:3]) and torch.equal(got[4:], out[4:])
    # one of the prefix: everyone's
    pool.k_scales[tables[0, 2].long()] = math.nan
    assert torch.isnan(share.attention(q, pool, tables, lengths, starts, found, max_new=1)).all()


def test_numbers_out_of_range_are_not_followed():
    """Prefixes of another step, tables and starts that make no sense: nothing outside is touched, and the next call is whole."""
    good = run([0] * 9, [200], [230] * 9, [1] * 9, heads=2, group=8, dim=64, block=16, max_new=1)
    q, pool, tables, starts, found, out, lse = good
    rng = random.Random(4)
    for _ in range(20):
        wild = i32([rng.choice([0, 1, 5, 9, -7, 2**31 - 1, -(2**31)]) for _ in range(10)])
        lengths = i32([rng.choice([0, 230, -1, 2**31 - 1, 5]) for _ in range(9)])
        other = torch.where(torch.rand(tables.shape, device="cuda") < 0.2, rng.choice([-1, 2**31 - 1, 0]), tables)
        bad = share.prefixes(other, lengths, wild, block_size=16, blocks=pool.blocks, tokens=9)
        share.attention(q, pool, other, lengths, wild, bad, max_new=1)
        share.attention(q, pool, tables, i32([230] * 9), starts, bad, max_new=1)
        share.attention(q, pool, other, lengths, wild, found, max_new=1)
        random_data = share.KVPrefixes(torch.randint(-(2**31), 2**31 - 1, found.data.shape, dtype=torch.int64, device="cuda").int(), 9, 9)
        share.attention(q, pool, tables, i32([230] * 9), starts, random_data, max_new=1)
    again, again_lse = share.attention(q, pool, tables, i32([230] * 9), starts, found, max_new=1, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)


def test_other_stream_and_graph():
    q, pool, tables, starts, found, out, lse = run([0] * 30, [300], [330] * 30, [1] * 30, heads=2, group=4, dim=64, block=32, max_new=1)
    lengths = i32([330] * 30)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = share.attention(q, pool, tables, lengths, starts, found, max_new=1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = share.prefixes(tables, lengths, starts, block_size=32, blocks=pool.blocks, tokens=30)
        held = share.attention(q, pool, tables, lengths, starts, step, max_new=1)
    lengths.fill_(320)
    q.copy_(torch.randn(q.shape, device="cuda").half())
    graph.replay()
    check_attention(q, pool, tables, [320] * 30, [1] * 30, held, None)


def test_refusals():
    q, pool, tables, starts, found, out, lse = run([0] * 3, [40], [50] * 3, [1] * 3, heads=2, group=2, dim=64, block=16, max_new=1)
    lengths = i32([50] * 3)
    for change, words in [(dict(shared=share.KVPrefixes(found.data, 3, 4)), "this step"), (dict(shared=share.KVPrefixes(found.data[:-1], 3, 3)), "this step"),
                          (dict(q=q[:, :3]), "multiple of kv_heads"), (dict(lengths=lengths.long()), "lengths"),
                          (dict(starts=starts[:-1]), "starts one more"), (dict(out=out[:2]), "out must"),
                          (dict(max_new=-1), ">= 0"), (dict(scale=math.inf), "finite"), (dict(q=q.float()), "float16")]:
        args = {**dict(q=q, pool=pool, tables=tables, lengths=lengths, starts=starts, shared=found), **change}
        with pytest.raises(ValueError, match=words):
            share.attention(**args)
    for change, words in [(dict(block_size=24), "block_size"), (dict(blocks=0), "blocks"), (dict(tokens=-1), "tokens"),
                          (dict(starts=starts[:-1]), "starts one more"), (dict(tables=tables.long()), "tables")]:
        args = {**dict(tables=tables, lengths=lengths, starts=starts, block_size=16, blocks=pool.blocks, tokens=3), **change}
        with pytest.raises(ValueError, match=words):
            share.prefixes(**args)
    empty = share.prefixes(tables[:0], lengths[:0], starts[:1], block_size=16, blocks=5, tokens=0)
    assert share.attention(q[:0], pool, tables[:0], lengths[:0], starts[:1], empty).shape == (0, 4, 64)


@pytest.mark.parametrize("members", [4, 30])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_negative_and_zero_scale(members, dtype):
    """Both kernels, whose signs are handled apart, and their join."""
    for scale in (-0.3, 0.0):
        run([0] * members, [300], [310 + 3 * i for i in range(members)], [1 + i % 2 for i in range(members)], heads=2, group=4, dim=64,
            block=16, dtype=dtype, scale=scale, max_new=2, grouped=sum(1 + i % 2 for i in range(members)))


def test_queries_of_any_strides():
    """Rows that are not 16-byte aligned are copied first; others are read where they are."""
    members, heads, dim = 20, 8, 64
    q, pool, tables, starts, found, out, lse = run([0] * members, [200], [230] * members, [1] * members, heads=2, group=4, dim=dim,
                                                   block=32, max_new=1)
    lengths = i32([230] * members)
    odd = torch.empty(members, heads, dim + 1, dtype=q.dtype, device="cuda")[..., 1:]
    flat = torch.empty(heads, members, dim, dtype=q.dtype, device="cuda").transpose(0, 1)
    for x in (odd, flat):
        x.copy_(q)
        assert torch.equal(share.attention(x, pool, tables, lengths, starts, found, max_new=1), out)


def test_two_streams_at_once():
    """Calls on two streams, each with its own prefixes and workspace, over one pool."""
    one = run([0] * 40, [3000], [3100] * 40, [1] * 40, heads=2, group=4, dim=128, block=64, max_new=1)
    q, pool, tables, starts, found, out, lse = one
    lengths, streams, got = i32([3100] * 40), [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, results in zip(streams, got):
            with torch.cuda.stream(stream):
                step = share.prefixes(tables, lengths, starts, block_size=64, blocks=pool.blocks, tokens=40)
                results.append(share.attention(q, pool, tables, lengths, starts, step, max_new=1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for results in got for x in results)


def test_hint_too_small():
    """max_new chooses kernels; a request that brings more than it says is right all the same."""
    groups, new = [0] * 12, [1] * 6 + [30] * 6
    run(groups, [500], [560 + i for i in range(12)], new, heads=2, group=4, dim=64, block=16, max_new=1, grouped=sum(new))


def test_largest_number_of_requests():
    requests = 8192
    tables = torch.arange(requests * 3, dtype=torch.int32, device="cuda").view(requests, 3)
    tables[:, 0] = tables[0, 0]
    tables[::2, 1] = tables[0, 1]
    starts = torch.arange(requests + 1, dtype=torch.int32, device="cuda")
    found = share.prefixes(tables, i32([48] * requests), starts, block_size=16, blocks=requests * 3, tokens=requests)
    # 8191 times one block, or 4095 times two: the longer of what saves the same is not taken, the one that saves more is
    assert (states(found) == 2).all()
    with pytest.raises(ValueError, match="8192"):
        share.prefixes(tables.repeat(2, 1), i32([48] * requests * 2), torch.arange(2 * requests + 1, dtype=torch.int32, device="cuda"),
                       block_size=16, blocks=requests * 3, tokens=2 * requests)
