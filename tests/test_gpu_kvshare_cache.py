"""SharedKVCache: plan, append, fork, compact, attention and materialize together, against lists of tokens.

Keys and values are whole numbers of which one in each token is 127, so that every scale is 1 and codes are exact: what is read
back is equal.  Attention's tolerance is that of tests/test_gpu_kvcache.py."""
from __future__ import annotations

import random
import sys
from pathlib import Path

import pytest
import torch

from test_gpu_kvcache import check_attention

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

share = pytest.importorskip("mlbricks_b200.kvshare")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def tokens_of(n, heads, dim):
    x = torch.randint(-126, 127, (n, heads, dim), device="cuda")
    x[..., 0] = 127
    return x.half()


class Model:
    def __init__(self, layers, requests, heads, dim):
        self.heads, self.dim, self.layers = heads, dim, layers
        self.rows = [[(torch.zeros(0, heads, dim, device="cuda").half(),) * 2 for _ in range(layers)] for _ in range(requests)]

    def held(self):
        return [row[0][0].shape[0] for row in self.rows]

    def fork(self, parents, keep):
        old = [list(row) for row in self.rows]
        for i, p in enumerate(parents):
            n = (keep[i] if keep else 1 << 30) if 0 <= p < len(old) else 0
            self.rows[i] = [(k[:n], v[:n]) for k, v in old[max(p, 0)]]

    def check(self, cache):
        held = self.held()
        assert cache.lengths.tolist() == held
        starts = torch.tensor([0] + held).cumsum(0).to(torch.int32).cuda()
        for layer in range(self.layers):
            k, v = cache.materialize(layer, starts, tokens=sum(held))
            assert torch.equal(k, torch.cat([row[layer][0] for row in self.rows]))
            assert torch.equal(v, torch.cat([row[layer][1] for row in self.rows]))
        used = {int(x) for i, n in enumerate(held) for x in cache.tables[i, :-(-n // cache.block_size)]}
        assert int(cache.ring[1] - cache.ring[0]) == cache.pools[0].blocks - len(used)


@pytest.mark.parametrize("block, heads, dim", [(16, 2, 32), (64, 1, 64)])
def test_any_order_of_calls(block, heads, dim):
    rng = random.Random(block)
    requests, layers, group = 9, 2, 3
    cache = share.SharedKVCache(layers, blocks=9 * 12, kv_heads=heads, head_dim=dim, requests=requests,
                                max_length=12 * block, block_size=block)
    model = Model(layers, requests, heads, dim)
    for step in range(40):
        kind = rng.choice(["step", "step", "step", "fork", "back", "compact", "free"])
        if kind == "compact":
            done = cache.compact()
            assert done.ring.tolist()[0] == 0
        elif kind in ("fork", "back", "free"):
            parents = [rng.choice([i, i, rng.randrange(requests)]) if kind != "free" else rng.choice([i, i, -1]) for i in range(requests)]
            keep = [rng.choice([1 << 30, max(n - rng.randrange(5), 0), n // 2]) for n in model.held()] if kind == "back" else None
            assert int(cache.fork(parents, keep).ring[2]) == 0
            model.fork(parents, keep)
        else:
            held = model.held()
            new = [rng.choice([-1, 0, 1, 1, 5, 2 * block + 1]) for _ in range(requests)]
            new = [min(n, 12 * block - h) for n, h in zip(new, held)]
            model.fork([-1 if n < 0 else i for i, n in enumerate(new)], None)
            if rng.random() < 0.5:
                plan = cache.plan(new)
            else:
                plan = cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), tokens=sum(max(n, 0) for n in new), max_new=max(new + [0]))
            assert int(plan.ring[2]) == 0
            count = sum(max(n, 0) for n in new)
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
                for options in ({}, {"window": 7}, {"first": torch.ones(requests, dtype=torch.int32, device="cuda")}):
                    out, lse = cache.attention(layer, q, return_lse=True, **options)
                    first = [1] * requests if "first" in options else None
                    check_attention(q, cache.pools[layer], cache.tables, model.held(), [max(n, 0) for n in new], out, lse,
                                    window=options.get("window", 0), first=first)
        model.check(cache)


def test_blocks_run_out():
    cache = share.SharedKVCache(1, blocks=4, kv_heads=1, head_dim=32, requests=4, max_length=64, block_size=16)
    cache.plan([20, 0, 0, 0])
    done = cache.fork([0, 0, 0, 0])  # two free blocks for three begun ones
    assert cache.lengths.tolist() == [20, 20, 20, 0] and done.ring.tolist() == [4, 4, 1, 2]
    assert cache.shares.tolist().count(2) == 1 and sum(cache.shares.tolist()) == 2
    cache.plan([-1, 0, 0, 0])  # its begun block is free, the shared one is not
    assert int(cache.ring[1] - cache.ring[0]) == 1 and sum(cache.shares.tolist()) == 1
    with pytest.raises(RuntimeError, match="plan"):
        cache.fork([0, 1, 2, 3])
        cache.attention(0, torch.zeros(1, 1, 32, device="cuda", dtype=torch.float16))


def test_captured_steps_between_forks():
    """A decode step captured once goes on after forks, compactions and releases made between its replays."""
    heads, dim, block, requests = 2, 64, 16, 6
    cache = share.SharedKVCache(1, blocks=80, kv_heads=heads, head_dim=dim, requests=requests, max_length=200, block_size=block)
    model = Model(1, requests, heads, dim)
    k, v = tokens_of(requests, heads, dim), tokens_of(requests, heads, dim)
    q = (0.01 * torch.randn(requests, 4 * heads, dim, device="cuda")).half()
    ones = torch.ones(requests, dtype=torch.int32, device="cuda")

    def step():
        cache.plan(ones, tokens=requests, max_new=1, releases=False)
        cache.append(0, k, v)
        return cache.attention(0, q)

    state = [t.clone() for t in (cache.lengths, cache.ring, cache.tables, cache.free, cache.shares)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for now, then in zip((cache.lengths, cache.ring, cache.tables, cache.free, cache.shares), state):
        now.copy_(then)

    def replay(times):
        for _ in range(times):
            k.copy_(tokens_of(requests, heads, dim)), v.copy_(tokens_of(requests, heads, dim))
            graph.replay()
            for i in range(requests):
                a, b = model.rows[i][0]
                model.rows[i][0] = (torch.cat([a, k[i:i + 1]]), torch.cat([b, v[i:i + 1]]))
            check_attention(q, cache.pools[0], cache.tables, model.held(), [1] * requests, out, None)
        model.check(cache)

    replay(35)
    for parents in ([0] * requests, [0, 0, 2, 2, 4, 4], [5, 4, 3, 2, 1, 0], [0, -1, 0, 3, -1, 3]):
        cache.fork(parents)
        model.fork(parents, None)
        replay(9)
        cache.compact()
        replay(3)


def test_samples_of_one_prompt():
    import kv_samples

    result = kv_samples.serve(steps=20)
    assert result["lengths"] == [333 + 20] * 6
    # the prompt's full blocks once, and for each sample the block that was begun and those behind it
    assert result["held"] == 333 // 32 + 6 * (-(-353 // 32) - 333 // 32)
    assert result["compacted"] == list(range(result["held"]))
    assert max(result["errors"]) < 0.05
