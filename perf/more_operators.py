"""The operators of requests that share cache blocks, and rotary positions, as cases that can be timed and compared.

Four operators that stand around the 8-bit paged key/value cache:

* `rotate` turns queries and keys by their positions: half and interleaved pairs, part of a head, frequencies
  scaled for long contexts;
* `fork` lets requests go on from what other requests hold: full blocks are shared and counted, a block that is
  still being filled is copied in every layer; it also rolls requests back and frees them;
* `compact` moves the blocks that requests hold to the front of the pool, in every layer;
* `attention` over requests whose tables begin alike reads what they share once for all of them.

`run` computes them from elementary torch operations in 32 bits (angles in 64), or, where `own` is true, with the
calls of `mlbricks_b200.rotary` and `mlbricks_b200.kvshare`.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
DEVICE = "cuda"


def listed():
    rotary = {"op": "rotate", "heads": 32, "kv": 8, "dim": 128, "part": 128, "interleaved": False, "scaling": "none",
              "dtype": "float16"}
    shared = {"op": "attention", "kv": 8, "group": 4, "dim": 128, "block": 64, "dtype": "float16", "groups": 1,
              "alone": 0.0, "new": 1, "lse": False}
    return [
        # A decode step of the BoltModel-shaped decoder: 8 requests, 12 heads over one, 32 wide.
        dict(rotary, name="rotate_step", tokens=8, heads=12, kv=1, dim=32, part=32, places=640),
        # The repository's three 2048-token prompts at the 8B stack's heads.
        dict(rotary, name="rotate_prompts", tokens=6144, places=2048, dtype="bfloat16"),
        # Odd heads of which part turns, in neighbouring pairs, 32 bits, far positions by a ramp of frequencies.
        dict(rotary, name="rotate_part", tokens=1001, heads=7, kv=7, dim=80, part=52, interleaved=True, scaling="ramp",
             places=131000, dtype="float32"),
        # Chunks of several long requests, positions far beyond those trained on, interpolated.
        dict(rotary, name="rotate_chunks", tokens=20000, places=100000, scaling="linear", interleaved=True),
        # Beam search in the BoltModel-shaped decoder: 4 requests of 4 beams choose their parents anew each step.
        {"name": "fork_beams", "op": "fork", "kind": "beams", "parents": 4, "each": 4, "prefix": 333, "own": 40,
         "layers": 3, "kv": 1, "dim": 32, "block": 32},
        # 31 samples of each of 4 prompts begin: every one copies a block that is begun, in 16 layers of 8 heads of 128.
        {"name": "fork_samples", "op": "fork", "kind": "samples", "parents": 4, "each": 32, "prefix": 1000, "own": 1,
         "layers": 16, "kv": 8, "dim": 128, "block": 128},
        # A small decoder's cache after many requests came and went.
        {"name": "compact_small", "op": "compact", "requests": 50, "groups": 2, "prefix": 300, "own": 400, "held": 0.5,
         "layers": 3, "kv": 1, "dim": 32, "block": 32},
        # The 8B stack's heads: 2900 blocks of which 60 % are held, two layers of it.
        {"name": "compact_large", "op": "compact", "requests": 60, "groups": 4, "prefix": 2100, "own": 3500, "held": 0.6,
         "layers": 2, "kv": 8, "dim": 128, "block": 64},
        # Four samples of one prompt in the BoltModel-shaped decoder.
        dict(shared, name="shared_small", requests=4, kv=1, group=12, dim=32, block=32, prefix=600, own=40),
        # A serving batch behind one system prompt of 8192 tokens at the 8B stack's heads.
        dict(shared, name="shared_batch", requests=64, prefix=8192, own=500, lse=True),
        # Five prompts with some samples each, others alone; heads of their own, several drafted tokens a step.
        dict(shared, name="shared_groups", requests=45, groups=5, alone=0.3, kv=16, group=1, dim=64, block=16,
             prefix=3000, own=700, new=5, dtype="bfloat16", lse=True),
        # The largest: four samples of one document of 131000 tokens.
        dict(shared, name="shared_long", requests=4, prefix=131000, own=300, dtype="bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "fork", "compact", "attention", "attention", "attention"])
    if op == "rotate":
        dim = rng.choice([32, 64, 80, 96, 128, 256, rng.randint(4, 130)])
        part = rng.choice([dim // 2 * 2, dim // 2 * 2, max(2, dim // 4 * 2), 2 * rng.randint(1, dim // 2)])
        heads = rng.choice([1, 3, 8, 12, 32, 64])
        kv = rng.choice([h for h in (1, 2, 3, 8) if h <= heads])
        return {"op": op, "tokens": _log(rng, 1, min(60_000, 100_000_000 // ((heads + kv) * dim))), "heads": heads, "kv": kv,
                "dim": dim, "part": part, "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "base", "ramp"]), "dtype": rng.choice(list(DTYPES)),
                "places": _log(rng, 16, 1_000_000)}
    block = rng.choice([16, 32, 64, 128])
    dim = rng.choice([32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "attention":
        requests, new = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5])
        prefix = _log(rng, 20, min(100_000, 250_000_000 // (requests * kv * dim)))
        return {"op": op, "requests": requests, "groups": rng.choice([1, 1, 2, 3, 7]), "alone": rng.choice([0.0, 0.0, 0.4]),
                "prefix": prefix, "own": _log(rng, 1, min(3000, 250_000_000 // (requests * kv * dim))), "new": new, "kv": kv,
                "group": rng.choice([1, 2, 4, 5, 8, 12]), "dim": dim, "block": block,
                "dtype": rng.choice(["float16", "bfloat16"]), "lse": rng.random() < 0.5}
    layers = rng.choice([1, 2, 3, 5, 8])
    room = max(600, 300_000_000 // (2 * layers * kv * dim))  # tokens that the pools may hold
    if op == "fork":
        parents, each = _log(rng, 1, 24), rng.choice([1, 2, 3, 4, 8, 16])
        own_ = _log(rng, 1, max(1, min(1000, room // (parents * each) // 4)))
        return {"op": op, "kind": rng.choice(["beams", "samples", "rollback"]), "parents": parents, "each": each,
                "prefix": _log(rng, 1, max(1, min(8000, room // parents // 2))), "own": own_, "layers": layers, "kv": kv,
                "dim": dim, "block": block}
    requests = _log(rng, 1, 300)
    return {"op": op, "requests": requests, "groups": rng.choice([1, 2, 5]),
            "prefix": _log(rng, 1, max(1, min(4000, room // 20))), "own": _log(rng, 1, max(1, min(4000, room // requests // 4))),
            "held": rng.choice([0.1, 0.5, 0.9]), "layers": layers, "kv": kv, "dim": dim, "block": block}


# ---- what a case holds: requests, what they share, tables -----------------------------------------------------


def _random(case):
    key = sum((i + 1) * v for i, v in enumerate(v for v in case.values() if type(v) is int))
    return torch.Generator().manual_seed(key)


def _requests(case):
    """The group of every request (-1: alone), the tokens that groups share, and what the requests hold behind them and
    bring, as host lists, from the case alone so that `work` knows them too.  The first group and the first request have
    the full lengths."""
    rng = _random(case)
    if case["op"] == "fork":
        requests, groups = case["parents"] * case["each"], case["parents"]
        group = [i // case["each"] for i in range(requests)]
    else:
        requests, groups = case["requests"], case["groups"]
        alone = torch.rand(requests, generator=rng) < case.get("alone", 0.0)
        # the members of a group are not neighbours
        group = [-1 if i and alone[i] else int(torch.randint(groups, (), generator=rng)) if i else 0 for i in range(requests)]
    part = torch.rand(groups, generator=rng, dtype=torch.float64)
    part[0] = 1.0
    prefix = (part * case["prefix"]).round().long().clamp(min=1).tolist()
    part = torch.rand(requests, 2, generator=rng, dtype=torch.float64)
    part[0] = 1.0
    behind = (part[:, 0] * case["own"]).round().long().tolist()
    new = (part[:, 1] * case.get("new", 0)).round().long().clamp(min=min(1, case.get("new", 0))).tolist()
    return group, prefix, behind, new


def _held(case):
    """Tokens that every request holds, new ones included; of `samples`, only the first of a group holds any yet."""
    group, prefix, behind, new = _requests(case)
    held = [(prefix[g] if g >= 0 else 0) + b + n for g, b, n in zip(group, behind, new)]
    if case["op"] == "fork" and case["kind"] == "samples":
        held = [h if i % case["each"] == 0 else 0 for i, h in enumerate(held)]
    return held


def _blocks(tokens, block):
    return -(-tokens // block)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _counts(case):
    """Of every request: its blocks, and how many of them it shares with its group; of every group: those blocks."""
    block = case["block"]
    group, prefix, _, _ = _requests(case)
    held = _held(case)
    mine = [_blocks(h, block) for h in held]
    common = [p // block for p in prefix]
    members = [sum(1 for g, h in zip(group, held) if g == k and h) for k in range(len(prefix))]
    common = [c if m > 1 else 0 for c, m in zip(common, members)]
    return mine, [common[g] if g >= 0 and m else 0 for g, m in zip(group, mine)], common, members, group


def _tables(case, total, rng):
    """A block table [requests, most blocks] over `total` shuffled blocks, -1 where a request has none; how often each
    block is shared; and the blocks that nobody holds."""
    mine, shared, common, members, group = _counts(case)
    order = torch.randperm(total, generator=rng, device=DEVICE).to(torch.int32)
    mine_t, shared_t = (torch.tensor(x, device=DEVICE) for x in (mine, shared))
    common_t = torch.tensor(common, device=DEVICE)
    group_at = common_t.cumsum(0) - common_t
    own_at = int(sum(common)) + (mine_t - shared_t).cumsum(0) - (mine_t - shared_t)
    column = torch.arange(max(1, max(mine)), device=DEVICE)[None]
    from_group = group_at[torch.tensor(group, device=DEVICE).clamp(min=0)][:, None] + column
    index = torch.where(column < shared_t[:, None], from_group, own_at[:, None] + column - shared_t[:, None])
    filled = column < mine_t[:, None]
    tables = torch.where(filled, order[index.clamp(max=total - 1)], -1).to(torch.int32)
    used = sum(common) + sum(m - s for m, s in zip(mine, shared))
    shares = torch.zeros(total, dtype=torch.int32, device=DEVICE)
    more = torch.tensor([max(m - 1, 0) for m in members], dtype=torch.int32, device=DEVICE)
    shares[order[:sum(common)].long()] = torch.repeat_interleave(more, common_t, output_size=sum(common))
    return tables.contiguous(), shares, order[used:]


def _used(case):
    mine, shared, common, _, _ = _counts(case)
    return sum(common) + sum(m - s for m, s in zip(mine, shared))


def _pools(case, blocks, layers, rng):
    """The layers' caches, one behind the other, as a running server holds them: codes, and a scale for each block and head."""
    shape = (layers, blocks, case["kv"], case["block"], case["dim"])
    pools = {}
    for side, size in (("k", 0.02), ("v", 0.015)):
        pools[side + "_codes"] = torch.randint(-127, 128, shape, generator=rng, device=DEVICE, dtype=torch.int8)
        pools[side + "_scales"] = size * torch.exp(0.5 * torch.randn(shape[:3], generator=rng, device=DEVICE))
    return pools


def _frequencies(case):
    """Angle of each pair at position 1, in 64 bits."""
    half = case["part"] // 2
    base, scaling, factor = 10000.0, case["scaling"], 8.0
    if scaling == "base" and half > 1:
        base *= factor ** (half / (half - 1))
    freq = base ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":  # pairs that turn seldom within the trained length are interpolated, the fast ones kept
        turns = 4096 * freq / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        freq = freq / factor * (1 - keep) + freq * keep
    return freq


def prepare(case, seed):
    rng = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    if op == "rotate":
        heads, kv, dim, tokens = case["heads"], case["kv"], case["dim"], case["tokens"]
        # queries and keys are views of a fused projection's output: queries, keys, values
        fused = torch.randn(tokens, heads + 2 * kv, dim, generator=rng, device=DEVICE).to(DTYPES[case["dtype"]])
        # prompts that run on, one after the other, each from a place of its own
        run_ = max(1, tokens // 3)
        first = torch.randint(case["places"], (4,), generator=rng, device=DEVICE)
        at = torch.arange(tokens, device=DEVICE)
        return {"case": case, "q": fused[:, :heads], "k": fused[:, heads:heads + kv], "frequencies": _frequencies(case),
                "positions": (first[(at // run_).clamp(max=3)] + at % run_).to(torch.int32)}
    block = case["block"]
    group, prefix, behind, new = _requests(case)
    held = _held(case)
    used = _used(case)
    if op == "attention":
        blocks = used + 3
        tables, _, _ = _tables(case, blocks, rng)
        fused = torch.randn(sum(new), (case["group"] + 2) * case["kv"], case["dim"], generator=rng, device=DEVICE)
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEVICE)
        return {"case": case, "tables": tables, "lengths": _int32(held), "starts": starts, "tokens": sum(new),
                "max_new": max(new), "max_length": max(held), "pools": _pools(case, blocks, 1, rng),
                "q": fused.mul_(2.5).to(DTYPES[case["dtype"]])[:, :case["group"] * case["kv"]]}
    requests = len(held)
    blocks = int(used / case["held"]) + 1 if op == "compact" else used + requests + 1
    tables, shares, unused = _tables(case, blocks, rng)
    if op == "fork":  # rows may come to hold as much as any other
        wide = torch.full((requests, tables.shape[1] + 1), -1, dtype=torch.int32, device=DEVICE)
        wide[:, :tables.shape[1]] = tables
        tables = wide
    head = blocks - min(blocks, 5)  # the ring's free part wraps
    free = torch.zeros(blocks, dtype=torch.int32, device=DEVICE)
    free[(head + torch.arange(len(unused), device=DEVICE)) % blocks] = unused
    state = {"case": case, "tables": tables, "shares": shares, "lengths": _int32(held), "free": free,
             "ring": torch.tensor([head, head + len(unused), 0, 0], dtype=torch.int64, device=DEVICE),
             "pools": _pools(case, blocks, case["layers"], rng)}
    if op == "fork":
        row = torch.arange(requests, device=DEVICE)
        each = case["each"]
        pick = torch.randint(each, (requests,), generator=rng, device=DEVICE)
        chance = torch.rand(requests, generator=rng, device=DEVICE)
        state["keep"] = None
        if case["kind"] == "beams":  # each beam goes on from a beam of its request; some requests are done
            done = (chance[row // each * each] < 0.2) & (row >= each)
            state["parents"] = torch.where(done, -1, row // each * each + pick).to(torch.int32)
        elif case["kind"] == "samples":  # the first row of each group holds the prompt
            state["parents"] = (row // each * each).to(torch.int32)
        else:  # drafted tokens that were not accepted are dropped, some requests are done
            state["parents"] = torch.where((chance < 0.1) & (row > 0), -1, row).to(torch.int32)
            state["keep"] = (state["lengths"] - (pick + 1) * (chance < 0.8)).clamp(min=0).to(torch.int32)
    return state


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


# ---- the plain forms ------------------------------------------------------------------------------------------


def _rotate_plain(s):
    case = s["case"]
    part, half = case["part"], case["part"] // 2
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:part:2], y[..., 1:part:2]
            pair = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:part]
            pair = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([pair, y[..., part:]], -1).to(x.dtype)

    return {"q": turned(s["q"]), "k": turned(s["k"])}


def _bump(counts, entries, mask, by):
    """counts[entry] += by for the entries of blocks that there are, where mask."""
    size = counts.shape[0]
    good = mask & (entries >= 0) & (entries < size)
    return counts.scatter_add_(0, entries.long().clamp(0, size - 1).flatten(), (good.int() * by).flatten())


def _copy_plain(pools, sources, targets):
    real = targets >= 0
    sources, targets = sources[real].long(), targets[real].long()
    for t in pools.values():
        t[:, targets] = t[:, sources]


def _fork_plain(s):
    block, tables, free, lengths = s["case"]["block"], s["tables"], s["free"], s["lengths"].long()
    requests, width = tables.shape
    size, room = free.shape[0], s["shares"].shape[0]
    row, column = torch.arange(requests, device=DEVICE), torch.arange(width, device=DEVICE)[None]
    parents = s["parents"].long()
    live = parents >= 0
    parent = parents.clamp(min=0)
    keep = torch.where(live, lengths[parent], 0)
    if s["keep"] is not None:
        keep = torch.minimum(keep, s["keep"].long())
    changed = ~((parents == row) & (keep == lengths))
    full, begun = keep // block, (keep % block > 0) & changed
    source = tables[parent]
    holders = s["shares"] + 1
    had = (lengths + block - 1) // block
    _bump(holders, tables, changed[:, None] & (column < had[:, None]), -1)
    _bump(holders, source, changed[:, None] & (column < full[:, None]), 1)
    tail = source[row, full.clamp(max=width - 1)].long()
    # of the rows that want a begun block, one keeps it, unless a row holds it whole
    key = row + torch.where(parents == row, 0, requests)
    first = torch.full((room,), 2 * requests, dtype=torch.int64, device=DEVICE)
    first.scatter_reduce_(0, tail.clamp(min=0), torch.where(begun, key, 2 * requests), "amin")
    keeps = begun & (holders[tail.clamp(min=0)] == 0) & (first[tail.clamp(min=0)] == key)
    need = begun & ~keeps
    before = need.cumsum(0) - need.long()
    avail = s["ring"][1] - s["ring"][0]
    got = need & (before < avail)
    refused = need & ~got
    _bump(holders, tail[:, None], keeps[:, None], 1)
    _bump(holders, source, (refused & changed)[:, None] & (column < full[:, None]), -1)
    fresh = free[(s["ring"][0] + before) % size]
    keep = torch.where(refused, 0, keep)
    out = torch.where(column < ((keep + block - 1) // block)[:, None], source, -1)
    out = torch.where(got[:, None] & (column == full[:, None]), fresh[:, None], out)
    gone = holders == 0
    place = torch.where(gone, (s["ring"][1] + gone.cumsum(0) - 1) % size, size)
    free.copy_(torch.cat([free, free[:1]]).scatter(0, place, torch.arange(room, device=DEVICE, dtype=torch.int32))[:size])
    at = torch.where(got, got.cumsum(0) - 1, requests)
    blank = torch.full((requests + 1,), -1, dtype=torch.int32, device=DEVICE)
    sources, targets = (blank.scatter(0, at, x.to(torch.int32))[:requests] for x in (tail, fresh))
    _copy_plain(s["pools"], sources, targets)
    copies = got.sum()
    ring = torch.stack([s["ring"][0] + copies, s["ring"][1] + gone.sum(), refused.sum(), copies])
    return {"lengths": keep.to(torch.int32), "tables": out, "shares": (holders - 1).clamp(min=0), "free": free,
            "ring": ring, "sources": sources, "targets": targets, "pools": s["pools"]}


def _compact_plain(s):
    block, tables = s["case"]["block"], s["tables"]
    blocks = s["shares"].shape[0]
    had = (s["lengths"].long() + block - 1) // block
    filled = torch.arange(tables.shape[1], device=DEVICE)[None] < had[:, None]
    held = _bump(torch.zeros_like(s["shares"]), tables, filled, 1) > 0
    count = held.sum()
    ids = torch.arange(blocks, device=DEVICE)
    high, low = held & (ids >= count), ~held & (ids < count)
    half = blocks // 2
    blank = torch.full((half + 1,), -1, dtype=torch.int64, device=DEVICE)
    sources, targets = (blank.scatter(0, torch.where(m, m.cumsum(0) - 1, half), ids)[:half] for m in (high, low))
    to = torch.cat([ids, ids[:1]]).scatter(0, torch.where(sources >= 0, sources, blocks), targets)[:blocks]
    shares = torch.zeros(blocks + 1, dtype=torch.int32, device=DEVICE)
    shares = shares.scatter(0, torch.where(held, to, blocks), s["shares"])[:blocks]
    _copy_plain(s["pools"], sources, targets)
    left = blocks - count
    return {"tables": torch.where(filled, to[tables.long().clamp(min=0)], -1).to(torch.int32), "shares": shares,
            "free": torch.where(ids < left, ids + count, -1).to(torch.int32),
            "ring": torch.stack([left * 0, left, left * 0, high.sum()]), "sources": sources.to(torch.int32),
            "targets": targets.to(torch.int32), "pools": s["pools"]}


def _attention_plain(s):
    case, pool = s["case"], {name: t[0] for name, t in s["pools"].items()}
    kv, group, dim, block = case["kv"], case["group"], case["dim"], case["block"]
    requests, new, columns = case["requests"], s["max_new"], _blocks(s["max_length"], block)
    tables = s["tables"][:, :columns].long().clamp(min=0)

    def side(name):
        x = pool[name + "_codes"][tables].float() * pool[name + "_scales"][tables][..., None, None]
        return x.transpose(1, 2).reshape(requests, kv, columns * block, dim)

    lengths, starts = s["lengths"].long(), s["starts"].long()
    counts = starts[1:] - starts[:-1]
    row = torch.arange(new, device=DEVICE)
    q = s["q"][(starts[:-1, None] + row).clamp(max=s["tokens"] - 1)].float()  # [requests, new, heads, dim]
    q = q.reshape(requests, new, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(requests, kv, group * new, dim)
    score = (q @ side("k").transpose(2, 3)).mul_(1 / math.sqrt(dim))
    place = (lengths - counts)[:, None] + row
    seen = torch.arange(columns * block, device=DEVICE) <= torch.minimum(place, lengths[:, None] - 1)[:, :, None]
    score = score.view(requests, kv, group, new, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(requests, kv, group * new, -1) @ side("v")).view(requests, kv, group, new, dim) / total
    request = torch.repeat_interleave(counts, output_size=s["tokens"])
    index = torch.arange(s["tokens"], device=DEVICE) - starts[request]
    out = out.permute(0, 3, 1, 2, 4)[request, index].reshape(s["tokens"], kv * group, dim).to(s["q"].dtype)
    if not case["lse"]:
        return out
    return out, (total.log() + top)[..., 0].permute(0, 3, 1, 2)[request, index].reshape(s["tokens"], kv * group)


_run_plain = {"rotate": _rotate_plain, "fork": _fork_plain, "compact": _compact_plain, "attention": _attention_plain}


# ---- the framework's calls ------------------------------------------------------------------------------------


def _own_pools(s):
    from mlbricks_b200 import kvcache
    return [kvcache.KVPool(*layer) for layer in zip(*(s["pools"][x] for x in ("k_codes", "k_scales", "v_codes", "v_scales")))]


def _rotate_own(s):
    from mlbricks_b200 import rotary
    q, k = rotary.rotate(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=s["case"]["interleaved"])
    return {"q": q, "k": k}


def _fork_own(s):
    from mlbricks_b200 import kvshare
    step = kvshare.fork(s["lengths"], s["tables"], s["shares"], s["free"], s["ring"], s["parents"],
                        block_size=s["case"]["block"], keep=s["keep"])
    kvshare.copy(_own_pools(s), step.moves)
    return {"lengths": step.lengths, "tables": step.tables, "shares": step.shares, "free": s["free"], "ring": step.ring,
            "sources": step.moves.sources, "targets": step.moves.targets, "pools": s["pools"]}


def _compact_own(s):
    from mlbricks_b200 import kvshare
    step = kvshare.compact(s["lengths"], s["tables"], s["shares"], block_size=s["case"]["block"])
    kvshare.copy(_own_pools(s), step.moves)
    return {"tables": step.tables, "shares": step.shares, "free": step.free, "ring": step.ring,
            "sources": step.moves.sources, "targets": step.moves.targets, "pools": s["pools"]}


def _attention_own(s):
    from mlbricks_b200 import kvshare
    pool = _own_pools(s)[0]
    shared = kvshare.prefixes(s["tables"], s["lengths"], s["starts"], block_size=pool.block_size, blocks=pool.blocks,
                              tokens=s["tokens"])
    return kvshare.attention(s["q"], pool, s["tables"], s["lengths"], s["starts"], shared, max_new=s["max_new"],
                             max_length=s["max_length"], return_lse=s["case"]["lse"])


_run_own = {"rotate": _rotate_own, "fork": _fork_own, "compact": _compact_own, "attention": _attention_own}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------


def _exact_rotate(case, s):
    out = {}
    part = case["part"]
    for name in ("q", "k"):
        x = s[name].double()
        y = x.clone()
        for i in range(part // 2):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + part // 2)
            turn = torch.polar(torch.ones_like(x[:, 0, 0]), s["positions"].double() * s["frequencies"][i])[:, None]
            pair = torch.complex(x[..., a], x[..., b]) * turn
            y[..., a], y[..., b] = pair.real, pair.imag
        out[name] = y
    return out


def _exact_attention(case, s):
    block, kv, group, dim = case["block"], case["kv"], case["group"], case["dim"]
    outs, lses, at, new = [], [], 0, _requests(case)[3]
    for r, (length, n) in enumerate(zip(_held(case), new)):
        ids = s["tables"][r, :_blocks(length, block)].long()
        k, v = (s["pools"][x + "_codes"][0, ids].double() * s["pools"][x + "_scales"][0, ids].double()[:, :, None, None] for x in ("k", "v"))
        k, v = (t.transpose(0, 1).reshape(kv, -1, dim)[:, :length] for t in (k, v))
        q = s["q"][at: at + n].double().view(n, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * n, dim)
        at += n
        hidden = torch.arange(length, device=DEVICE)[None] > length - n + torch.arange(n, device=DEVICE)[:, None]
        score = (q @ k.transpose(1, 2) / math.sqrt(dim)).masked_fill(hidden.repeat(group, 1), -math.inf)
        lse = torch.logsumexp(score, 2)
        out = torch.exp(score - lse[:, :, None]) @ v
        outs.append(out.view(kv, group, n, dim).permute(2, 0, 1, 3).reshape(n, kv * group, dim))
        lses.append(lse.view(kv, group, n).permute(2, 0, 1).reshape(n, kv * group))
    out = torch.cat(outs)
    return (out, torch.cat(lses)) if case["lse"] else out


def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits.  Forks and compactions choose and copy: none of it is computed."""
    if case["op"] in ("fork", "compact"):
        return None
    return (_exact_rotate if case["op"] == "rotate" else _exact_attention)(case, prepare(case, seed))


def work(case):
    op = case["op"]
    if op == "rotate":
        size = DTYPES[case["dtype"]].itemsize
        elements = case["tokens"] * (case["heads"] + case["kv"])
        return {"bytes": 2 * size * elements * case["dim"] + 4 * case["tokens"] + 4 * case["part"],
                "flops": 3 * elements * case["part"]}
    block, kv, dim = case["block"], case["kv"], case["dim"]
    mine, shared, common, members, group = _counts(case)
    if op == "attention":
        prefix, new, held = _requests(case)[1], _requests(case)[3], _held(case)
        # every held token once, what groups share once for all of them
        keys = sum(h - s * block for h, s in zip(held, shared)) + sum(common) * block
        heads, row = kv * case["group"], 2 * kv * dim
        pairs = sum(n * (h - n) + n * (n + 1) // 2 for n, h in zip(new, held))
        return {"bytes": keys * (row + (8 * kv + 4) / block) + sum(new) * heads * (4 * dim + (4 if case["lse"] else 0)),
                "flops": 4 * pairs * heads * dim}
    requests, used = len(mine), _used(case)
    if op == "fork":
        blocks, held, each = used + requests + 1, _held(case), case["each"]
        if case["kind"] == "samples":
            begun = [h % block > 0 for h in held]
            copies = sum((each - 1) * begun[p * each] for p in range(case["parents"]))
        elif case["kind"] == "beams":  # of the beams that go on, those that are not the first of their parent
            copies = 0.85 * requests * ((1 - 1 / each) ** each) * (1 - 1 / block)
        else:
            copies = 0.0
        tables = 8 * requests * (max(mine) + 1)
    else:
        blocks = int(used / case["held"]) + 1
        copies = used * (blocks - used) / blocks
        tables = 8 * sum(mine)
    moved = 4 * case["layers"] * kv * (block * dim + 4)  # keys and values, read and written
    return {"bytes": copies * moved + tables + 8 * blocks + 8 * requests, "flops": 0}
