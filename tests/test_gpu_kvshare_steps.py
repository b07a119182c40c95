"""SharedKVCache where its attention reads prefixes once: capacities at which ``takes_prefixes`` says yes, so that the
prefixes of a step are found, kept over its layers, dropped by what comes between steps, and captured.

Keys and values are exact, and attention's tolerance is that of tests/test_gpu_kvcache.py, as in
tests/test_gpu_kvshare_cache.py and tests/test_gpu_kvshare_attention.py."""
from __future__ import annotations

import random

import pytest
import torch

from test_gpu_kvcache import check_attention
from test_gpu_kvshare_attention import states
from test_gpu_kvshare_cache import Model, tokens_of

pytestmark = pytest.mark.gpu

share = pytest.importorskip("mlbricks_b200.kvshare")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def grouped(cache):
    """Tokens of the step that are in a group."""
    return 0 if cache._shared is None else int((states(cache._shared) == 2).sum())


def sharers(rows, new, block):
    """Is there a pair of rows that bring tokens and hold the same first block ahead of them?  (Rows as of Model's first layer:
    equal beginnings are shared blocks here, since every token is drawn afresh.)"""
    firsts = [bytes(row[0][0][:block].cpu().numpy().tobytes()) for row, n in zip(rows, new) if n > 0 and row[0][0].shape[0] >= block]
    return len(firsts) - len(set(firsts))


@pytest.mark.parametrize("block, heads, dim, group", [(16, 2, 32, 3), (64, 1, 64, 12), (32, 1, 128, 4)])
def test_any_order_of_calls(block, heads, dim, group):
    rng = random.Random(block)
    requests, layers, most = 9, 2, 12 * block
    cache = share.SharedKVCache(layers, blocks=9 * 12, kv_heads=heads, head_dim=dim, requests=requests, max_length=150_000,
                                block_size=block)
    pool = cache.pools[0]
    model = Model(layers, requests, heads, dim)
    shared_steps = 0
    for step in range(40):
        kind = rng.choice(["step", "step", "step", "fork", "back", "compact", "prompts"]) if step else "prompts"
        if kind == "compact":
            cache.compact()
            assert cache._shared is None
        elif kind in ("fork", "back"):
            parents = [rng.choice([i, i, rng.randrange(requests)]) for i in range(requests)]
            keep = [rng.choice([1 << 30, max(n - rng.randrange(5), 0)]) for n in model.held()] if kind == "back" else None
            assert int(cache.fork(parents, keep).ring[2]) == 0
            assert cache._shared is None
            model.fork(parents, keep)
        else:
            held = model.held()
            if kind == "prompts":  # of rows that hold nothing, or a few decode steps for the others
                new = [2 * block + i if held[i] == 0 else rng.choice([0, 1]) for i in range(requests)]
            else:
                new = [-1 if rng.random() < 0.04 else rng.choice([0, 1, 1, 1, 3]) for i in range(requests)]
            new = [min(n, most - h) for n, h in zip(new, held)]
            model.fork([-1 if n < 0 else i for i, n in enumerate(new)], None)
            ahead = sharers(model.rows, new, block)
            as_tensor = torch.tensor(new, dtype=torch.int32, device="cuda")
            count = sum(max(n, 0) for n in new)
            plan = cache.plan(new) if rng.random() < 0.5 else cache.plan(as_tensor, tokens=count, max_new=max(new + [0]))
            assert int(plan.ring[2]) == 0 and cache._shared is None
            takes = share.takes_prefixes(pool, heads * group, requests, count, max(new + [0]), cache.max_length)
            assert takes == (max(new + [0]) * group < 49)
            for layer in range(layers):
                k, v = tokens_of(count, heads, dim), tokens_of(count, heads, dim)
                cache.append(layer, k, v)
                at = 0
                for i, n in enumerate(new):
                    if n > 0:
                        a, b = model.rows[i][layer]
                        model.rows[i][layer] = (torch.cat([a, k[at:at + n]]), torch.cat([b, v[at:at + n]]))
                        at += n
                q = (0.01 * torch.randn(count, heads * group, dim, device="cuda")).half()
                before = cache._shared
                out, lse = cache.attention(layer, q, return_lse=True)
                assert (cache._shared is not None) == takes and (before is None or before is cache._shared)
                check_attention(q, cache.pools[layer], cache.tables, model.held(), [max(n, 0) for n in new], out, lse)
            if takes:
                assert (grouped(cache) > 0) == (ahead > 0)
                shared_steps += ahead > 0
        model.check(cache)
    assert shared_steps >= 8


def test_captured_steps_between_forks():
    """As in tests/test_gpu_kvshare_cache.py, with prefixes that the captured step finds anew in every replay, and two layers
    that read them."""
    heads, dim, block, requests, layers = 2, 64, 16, 6, 2
    cache = share.SharedKVCache(layers, blocks=80, kv_heads=heads, head_dim=dim, requests=requests, max_length=40_000,
                                block_size=block)
    assert share.takes_prefixes(cache.pools[0], 4 * heads, requests, requests, 1, cache.max_length)
    model = Model(layers, requests, heads, dim)
    k, v = ([tokens_of(requests, heads, dim) for _ in range(layers)] for _ in "kv")
    q = (0.01 * torch.randn(requests, 4 * heads, dim, device="cuda")).half()
    ones = torch.ones(requests, dtype=torch.int32, device="cuda")

    def step():
        cache.plan(ones, tokens=requests, max_new=1, releases=False)
        outs = []
        for layer in range(layers):
            cache.append(layer, k[layer], v[layer])
            outs.append(cache.attention(layer, q))
        return outs

    state = [t.clone() for t in (cache.lengths, cache.ring, cache.tables, cache.free, cache.shares)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for now, then in zip((cache.lengths, cache.ring, cache.tables, cache.free, cache.shares), state):
        now.copy_(then)
    found = cache._shared  # the graph's

    def replay(times, members):
        for _ in range(times):
            for layer in range(layers):
                k[layer].copy_(tokens_of(requests, heads, dim)), v[layer].copy_(tokens_of(requests, heads, dim))
            graph.replay()
            for layer in range(layers):
                for i in range(requests):
                    a, b = model.rows[i][layer]
                    model.rows[i][layer] = (torch.cat([a, k[layer][i:i + 1]]), torch.cat([b, v[layer][i:i + 1]]))
                check_attention(q, cache.pools[layer], cache.tables, model.held(), [1] * requests, outs[layer], None)
            assert int((states(found) == 2).sum()) == members
        model.check(cache)

    replay(35, 0)
    for parents, members in (([0] * requests, 6), ([0, 0, 2, 2, 4, 4], 6), ([5, 4, 3, 2, 1, 0], 6)):
        cache.fork(parents)
        model.fork(parents, None)
        replay(9, members)
        cache.compact()
        replay(3, members)
    cache.fork([0, 1, -1, -1, -1, -1])
    model.fork([0, 1, -1, -1, -1, -1], None)
    replay(3, 2)


def forked(requests=7, heads=1, dim=64, block=16):
    """A cache whose rows all share a prompt of five blocks and some, and one step of a token each behind it."""
    cache = share.SharedKVCache(1, blocks=60, kv_heads=heads, head_dim=dim, requests=requests, max_length=70_000, block_size=block)
    cache.plan([5 * block + 3] + [0] * (requests - 1))
    cache.append(0, tokens_of(5 * block + 3, heads, dim), tokens_of(5 * block + 3, heads, dim))
    cache.fork([0] * requests)
    cache.plan([1] * requests)
    cache.append(0, tokens_of(requests, heads, dim), tokens_of(requests, heads, dim))
    return cache


def test_fewer_queries_than_the_step_has():
    """Queries of the step's first requests only, and of all of them, in one step: as KVCache allows."""
    cache = forked()
    q = (0.01 * torch.randn(7, 4, 64, device="cuda")).half()
    for n in (7, 5, 7, 2):
        out, lse = cache.attention(0, q[:n].contiguous(), return_lse=True)
        assert grouped(cache) == n
        check_attention(q[:n], cache.pools[0], cache.tables, cache.lengths.tolist(), [1] * n + [0] * (7 - n), out, lse)


def test_a_refused_plan_frees_nothing():
    """Calls of `plan` that are refused leave the rows that they would have released as they were."""
    cache = forked()
    state = [cache.lengths, cache.tables, cache.shares, cache.free, cache.ring]
    before = [t.clone() for t in state]
    ints = torch.tensor([-1, 1, -1, 1, 1, 1, 1], dtype=torch.int32, device="cuda")
    for args, options in [((ints,), {}), ((ints.long(),), dict(tokens=5)), ((ints,), dict(tokens=-1)),
                          ((ints.float(),), dict(tokens=5)), ((ints[:6],), dict(tokens=5)), ((ints[:1],), dict(tokens=5)),
                          ((ints.repeat(2)[::2],), dict(tokens=5)), ((ints.cpu(),), dict(tokens=5)),
                          (([-1, 1],), {}), (([-1] * 8,), {}), (([-1] + [2**31] + [1] * 5,), {})]:
        with pytest.raises((ValueError, RuntimeError)):
            cache.plan(*args, **options)
        assert all(torch.equal(a, b) for a, b in zip(state, before)), (args, options)
    assert cache.plan(ints.view(7, 1), tokens=5, max_new=1).ring.tolist()[2] == 0
    assert cache.lengths.tolist() == [0, 85, 0, 85, 85, 85, 85]
