"""The operators of the 8-bit paged key/value cache, as cases that can be timed and compared.

Four operators belong together: `plan` gives every request its cache blocks and every new token
its slot, `append` quantises the new keys and values into those slots, `attention` reads the
cache, and `materialize` turns parts of it back into 16-bit keys and values.  A cache block holds
`block` tokens of one head as signed 8-bit codes under one 32-bit scale; value = code * scale.

`run` computes them from elementary torch operations in 32 bits, or, where `own` is true, with
the calls of `mlbricks_b200.kvcache`.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
DEVICE = "cuda"


def listed():
    step = {"op": "attention", "kv": 8, "group": 4, "dim": 128, "block": 64, "dtype": "float16",
            "window": 0, "lse": False}
    return [
        # One decode step of 64 requests: one token each, some finished, some at a block's edge.
        {"name": "plan_step", "op": "plan", "requests": 64, "past": 8192, "new": 1, "done": 0.1, "spare": 1.0,
         "block": 64},
        # Admission of ragged prompts next to running requests, with the smallest blocks.
        {"name": "plan_prompts", "op": "plan", "requests": 1000, "past": 700, "new": 250, "done": 0.05, "spare": 1.0,
         "block": 16},
        # One decode step's keys and values of the 8B stack (8 heads of 128): one token each into partial blocks.
        {"name": "append_step", "op": "append", "requests": 64, "past": 4000, "new": 1, "kv": 8, "dim": 128,
         "block": 64, "dtype": "float16"},
        # Prompt chunks of ragged lengths, behind odd pasts, views of a fused projection.
        {"name": "append_prompts", "op": "append", "requests": 21, "past": 777, "new": 3001, "kv": 8, "dim": 128,
         "block": 16, "dtype": "bfloat16"},
        # What the one shared head of the BoltModel-shaped decoder holds (384 / 12 = 32 wide): 8 requests of up to 640.
        {"name": "materialize_shared", "op": "materialize", "requests": 8, "length": 640, "kv": 1, "dim": 32,
         "block": 32, "dtype": "float16"},
        # Long requests handed on whole.
        {"name": "materialize_long", "op": "materialize", "requests": 16, "length": 8000, "kv": 8, "dim": 128,
         "block": 64, "dtype": "float16"},
        # The smallest attention: a decode step of the BoltModel-shaped decoder, 12 heads over one, batch 8.
        dict(step, name="step_shared", requests=8, past=600, new=1, kv=1, group=12, dim=32, block=32),
        # A serving batch's decode step at the 8B stack's heads: 64 requests of 1 to 8192 tokens.
        dict(step, name="step_batch", requests=64, past=8191, new=1, lse=True),
        # A decode step of one long request, 131071 tokens: the work has to be split over the length.
        dict(step, name="step_long", requests=1, past=131070, new=1, dtype="bfloat16"),
        # Prompts of ragged odd lengths from nothing, 64 wide heads of their own, a sliding window.
        dict(step, name="prompts_window", requests=12, past=0, new=1900, kv=16, group=1, dim=64, block=16, window=500),
        # The repository's 2048-token prompts at the 8B stack's heads, behind short pasts.
        dict(step, name="prompts", requests=3, past=99, new=2048, lse=True),
        # The largest: a chunk of 4096 tokens behind 12000.
        dict(step, name="chunk_long", requests=1, past=12000, new=4096, dtype="bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["plan", "append", "materialize", "attention", "attention", "attention"])
    block = rng.choice([16, 32, 64, 128])
    if op == "plan":
        requests = _log(rng, 1, 1500)
        return {"op": op, "requests": requests, "past": _log(rng, 1, min(8192, 1_000_000 // requests)),
                "new": _log(rng, 1, 250_000 // requests), "done": rng.choice([0.0, 0.1, 0.3]),
                "spare": rng.choice([1.0, 1.0, 0.6]), "block": block}
    dtype = rng.choice(list(DTYPES))
    dim = rng.choice([32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "append":
        requests = _log(rng, 1, 128)
        most = 1 if rng.random() < 0.4 else min(8000, 30_000_000 // (requests * kv * dim))
        return {"op": op, "requests": requests, "past": _log(rng, 1, 2000), "new": _log(rng, 1, most), "kv": kv,
                "dim": dim, "block": block, "dtype": dtype}
    if op == "materialize":
        requests = _log(rng, 1, 64)
        return {"op": op, "requests": requests, "length": _log(rng, 1, min(20_000, 60_000_000 // (requests * kv * dim))),
                "kv": kv, "dim": dim, "block": block, "dtype": dtype}
    group = rng.choice([1, 2, 4, 5, 8, 12])
    window = rng.choice([0, 0, 0, _log(rng, 16, 3000)])
    if rng.random() < 0.55:  # steps of one or a few tokens behind pasts of any length
        requests, new = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5])
        past = _log(rng, 1, min(131_000, 250_000_000 // (requests * kv * dim)))
    else:  # prompts and chunks
        new = _log(rng, 6, 3500)
        past = rng.choice([0, _log(rng, 1, 10_000)])
        requests = rng.randint(1, max(1, min(12, int(1.6e9 / (new * (past + new) * kv * group)))))
    return {"op": op, "requests": requests, "past": past, "new": new, "kv": kv, "group": group, "dim": dim,
            "block": block, "dtype": dtype, "window": window, "lse": rng.random() < 0.5}


def _lengths(case):
    """What the requests hold and what they bring (host lists), from the case alone so that `work` knows them too.
    The first request has the full lengths, the others anything down to nothing, or to one new token."""
    key = sum((i + 1) * v for i, v in enumerate(v for v in case.values() if type(v) is int))
    rng = torch.Generator().manual_seed(key)
    part = torch.rand(case["requests"], 2, generator=rng, dtype=torch.float64)
    part[0] = 1.0
    if case["op"] == "materialize":  # the tokens from `past` on, `new` of them
        total = (part[:, 0] * case["length"]).round().long()
        past = torch.where(part[:, 1] < 0.3, total // 3, torch.zeros_like(total))
        return past.tolist(), (total - past).tolist()
    past = (part[:, 0] * case["past"]).round().long()
    new = (part[:, 1] * case["new"]).round().long().clamp(min=1)
    if case["op"] == "plan":
        done = torch.rand(case["requests"], generator=rng) < case["done"]
        new = torch.where(done, torch.full_like(new, -1), new)
    return past.tolist(), new.tolist()


def _blocks(tokens, block):
    return -(-tokens // block)


def _starts(counts):
    return torch.tensor([0] + counts, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEVICE)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(held, block, spare, rng):
    """A block table [requests, most blocks] of shuffled blocks, -1 where a request has none, and the blocks left over."""
    counts = torch.tensor([_blocks(h, block) for h in held], device=DEVICE)
    total = int(counts.sum())
    order = torch.randperm(total + spare, generator=rng, device=DEVICE).to(torch.int32)
    width = max(1, int(counts.max()))
    index = torch.arange(width, device=DEVICE)[None] + (counts.cumsum(0) - counts)[:, None]
    filled = torch.arange(width, device=DEVICE)[None] < counts[:, None]
    tables = torch.where(filled, order[index.clamp(max=total + spare - 1)], torch.full_like(index, -1, dtype=torch.int32))
    return tables.contiguous(), order[total:]


def _pool(case, blocks, rng):
    """A cache of `blocks` blocks as a running server holds it: codes in a bell shape, a scale for each block and head."""
    shape = (blocks, case["kv"], case["block"], case["dim"])
    pool = {}
    for side, size in (("k", 0.02), ("v", 0.015)):
        codes = torch.randn(shape, generator=rng, device=DEVICE, dtype=torch.float16)
        pool[side + "_codes"] = codes.mul_(40).round_().clamp_(-127, 127).to(torch.int8)
        pool[side + "_scales"] = size * torch.exp(0.5 * torch.randn(shape[:2], generator=rng, device=DEVICE))
    return pool


def prepare(case, seed):
    rng = torch.Generator(device=DEVICE).manual_seed(seed)
    past, new = _lengths(case)
    block = case["block"]
    if case["op"] == "plan":
        wanted = [_blocks(p + max(n, 0), block) for p, n in zip(past, new)]
        more = sum(w - _blocks(p, block) for w, p in zip(wanted, past))
        room = max(1, int(more * case["spare"]))  # blocks that are free
        tables, unused = _tables(past, block, room + 1, rng)
        grown = torch.full((len(past), max(1, max(wanted))), -1, dtype=torch.int32, device=DEVICE)
        grown[:, : tables.shape[1]] = tables[:, : grown.shape[1]]
        size = sum(_blocks(p, block) for p in past) + room + 1
        head = size - min(size, 5)  # the ring's free part wraps
        free = torch.zeros(size, dtype=torch.int32, device=DEVICE)
        free[(head + torch.arange(room, device=DEVICE)) % size] = unused[:room]
        return {"case": case, "past": _int32(past), "new": _int32(new), "tables": grown, "free": free,
                "ring": torch.tensor([head, head + room, 0, 0], dtype=torch.int64, device=DEVICE),
                "tokens": sum(max(n, 0) for n in new),
                "released": sum(_blocks(p, block) for p, n in zip(past, new) if n < 0)}
    held = [p + n for p, n in zip(past, new)]
    tables, _ = _tables(held, block, 3, rng)
    blocks = sum(_blocks(h, block) for h in held) + 3
    state = {"case": case, "tables": tables, "lengths": _int32(held), "new": _int32(new), "past": _int32(past),
             "starts": _starts(new), "tokens": sum(new), "max_new": max(new), "max_length": max(held),
             **_pool(case, blocks, rng)}
    tokens, dtype = state["tokens"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        request, place = _tokens(state)
        state["slots"] = tables[request, place // block].long() * block + place % block
        # the keys and values are views of a fused projection's output: queries, keys, values
        fused = torch.randn(tokens, 6 * case["kv"], case["dim"], generator=rng, device=DEVICE, dtype=torch.float32)
        fused *= torch.exp(0.4 * torch.randn(1, 6 * case["kv"], case["dim"], generator=rng, device=DEVICE))
        fused = fused.to(dtype)
        state["k"], state["v"] = fused[:, 4 * case["kv"]: 5 * case["kv"]], fused[:, 5 * case["kv"]:]
        # what is read back: every block that the call touches
        first = [p // block * block for p in past]
        state["first"] = _int32(first)
        state["back"] = sum(h - f for h, f in zip(held, first))
        state["back_starts"] = _starts([h - f for h, f in zip(held, first)])
    elif case["op"] == "attention":
        heads = case["kv"] * case["group"]
        fused = torch.randn(tokens, heads + 2 * case["kv"], case["dim"], generator=rng, device=DEVICE,
                            dtype=torch.float32).mul_(2.5).to(dtype)
        state["q"] = fused[:, :heads]
    return state


def _tokens(state):
    """Request and position of every new token."""
    request = torch.repeat_interleave(state["new"].clamp(min=0), output_size=state["tokens"])
    index = torch.arange(state["tokens"], device=request.device)
    return request, state["past"][request].long() + index - state["starts"][request].long()


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


# ---- the plain forms ------------------------------------------------------------------------------------------


def _plan_plain(s):
    block, tables, free = s["case"]["block"], s["tables"], s["free"]
    past, new = s["past"].long(), s["new"].long()
    head, tail = s["ring"][0], s["ring"][1]
    width, size = tables.shape[1], free.shape[0]
    add = new.clamp(min=0)
    had = (past + block - 1) // block
    wanted = (past + add + block - 1) // block - had
    wide = had + wanted > width
    need = torch.where(wide, 0, wanted)
    before = need.cumsum(0) - need
    fits = (new >= 0) & ~wide & ((need == 0) | (before + need <= tail - head))
    ends = add.cumsum(0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    request = torch.repeat_interleave(add, output_size=s["tokens"])
    place = past[request] + torch.arange(s["tokens"], device=past.device) - starts[request]
    column = place // block
    fresh = column - had[request]
    inside = column.clamp(max=width - 1)
    old = tables[request, inside]
    taken = free[(head + before[request] + fresh.clamp(min=0)) % size]
    ok = fits[request]
    entry = torch.where(ok & (fresh >= 0), taken, old)
    slots = torch.where(ok, entry.long() * block + place % block, -1)
    gone = torch.where(new < 0, had, 0)
    gone_request = torch.repeat_interleave(gone, output_size=s["released"])
    order = torch.arange(s["released"], device=past.device)
    given = tables[gone_request, order - (gone.cumsum(0) - gone)[gone_request]]
    free[(tail + order) % size] = given
    tables[request, inside] = entry
    ring = torch.stack([head + torch.where(fits, before + need, 0).max(), tail + gone.sum(),
                        torch.where(fits, 0, wanted).sum(), ends[-1]])
    return {"lengths": torch.where(new < 0, 0, torch.where(fits, past + add, past)).int(), "starts": starts.int(),
            "slots": slots, "positions": place.int(), "ring": ring, "tables": tables, "free": free}


def _append_side_plain(s, x, codes, scales):
    block = codes.shape[2]
    x, slots = x.float(), s["slots"]
    where, offset = slots // block, slots % block
    # the largest size among the new tokens of each block and head
    most = torch.zeros_like(scales).index_reduce_(0, where, x.abs().amax(2), "amax")
    # a request's first new token may find its block begun: what is there keeps its scale, or moves to the larger one
    begun = slots[s["starts"][:-1].long()]
    mine, kept = begun // block, begun % block
    old_scale = torch.where((kept > 0)[:, None], scales[mine], 0)
    fresh = torch.where(most.isfinite(), most, math.nan) / torch.tensor(127.0, device=x.device)
    fresh[mine] = torch.maximum(fresh[mine], old_scale)
    old = codes[mine]
    ratio = torch.where(fresh[mine] > old_scale, old_scale / fresh[mine], 1.0)
    moved = (old.float() * ratio[:, :, None, None]).round().to(torch.int8)
    mask = torch.arange(block, device=x.device)[None, :] < kept[:, None]
    codes[mine] = torch.where(mask[:, None, :, None], moved, old)
    scales.index_copy_(0, where, fresh[where])
    unit = fresh[where][:, :, None]
    codes[where, :, offset] = torch.where(unit > 0, x / unit, 0).round().clamp(-127, 127).to(torch.int8)


def _append_plain(s):
    _append_side_plain(s, s["k"], s["k_codes"], s["k_scales"])
    _append_side_plain(s, s["v"], s["v_codes"], s["v_scales"])
    back = _materialize_tokens(s, s["first"], s["back_starts"], s["back"])
    return {**back, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _materialize_tokens(s, first, starts, tokens):
    block, dtype = s["case"]["block"], DTYPES[s["case"]["dtype"]]
    request = torch.repeat_interleave(starts[1:] - starts[:-1], output_size=tokens)
    place = first[request].long() + torch.arange(tokens, device=request.device) - starts[request].long()
    where = s["tables"][request, place // block].long()
    return {side: (s[side + "_codes"][where, :, place % block].float() * s[side + "_scales"][where][:, :, None]).to(dtype)
            for side in ("k", "v")}


def _materialize_plain(s):
    return _materialize_tokens(s, s["past"], s["starts"], s["tokens"])


def _attention_plain(s):
    case = s["case"]
    kv, group, dim, block = case["kv"], case["group"], case["dim"], case["block"]
    requests, new, columns = case["requests"], s["max_new"], _blocks(s["max_length"], block)
    tables = s["tables"][:, :columns].long().clamp(min=0)

    def side(name):
        x = s[name + "_codes"][tables].float() * s[name + "_scales"][tables][..., None, None]
        return x.transpose(1, 2).reshape(requests, kv, columns * block, dim)

    lengths, starts = s["lengths"].long(), s["starts"].long()
    counts = starts[1:] - starts[:-1]
    row = torch.arange(new, device=tables.device)
    q = s["q"][(starts[:-1, None] + row).clamp(max=s["tokens"] - 1)].float()  # [requests, new, heads, dim]
    q = q.reshape(requests, new, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(requests, kv, group * new, dim)
    score = (q @ side("k").transpose(2, 3)).mul_(1 / math.sqrt(dim))
    place = (lengths - counts)[:, None] + row  # [requests, new]
    key = torch.arange(columns * block, device=tables.device)
    seen = (key <= place[:, :, None]) & (key < lengths[:, None, None])
    if case["window"]:
        seen &= key > place[:, :, None] - case["window"]
    score = score.view(requests, kv, group, new, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top.isfinite(), top, 0)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = weight.view(requests, kv, group * new, -1) @ side("v")
    out = out.view(requests, kv, group, new, dim) / torch.where(total > 0, total, 1)
    request = torch.repeat_interleave(counts, output_size=s["tokens"])
    index = torch.arange(s["tokens"], device=tables.device) - starts[request]
    out = out.permute(0, 3, 1, 2, 4)[request, index].reshape(s["tokens"], kv * group, dim).to(s["q"].dtype)
    if not case["lse"]:
        return out
    lse = (total.log() + top)[..., 0].permute(0, 3, 1, 2)[request, index].reshape(s["tokens"], kv * group)
    return out, lse


_run_plain = {"plan": _plan_plain, "append": _append_plain, "materialize": _materialize_plain,
              "attention": _attention_plain}


# ---- the framework's calls ------------------------------------------------------------------------------------


def _kvcache():
    from mlbricks_b200 import kvcache
    return kvcache


def _own_pool(s):
    return _kvcache().KVPool(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])


def _plan_own(s):
    step = _kvcache().plan(s["past"], s["new"], s["tables"], s["free"], s["ring"], block_size=s["case"]["block"],
                           tokens=s["tokens"])
    return {"lengths": step.lengths, "starts": step.starts, "slots": step.slots, "positions": step.positions,
            "ring": step.ring, "tables": s["tables"], "free": s["free"]}


def _append_own(s):
    pool = _own_pool(s)
    _kvcache().append(s["k"], s["v"], pool, s["slots"])
    k, v = _kvcache().materialize(pool, s["tables"], s["back_starts"], first=s["first"], tokens=s["back"],
                                  dtype=DTYPES[s["case"]["dtype"]])
    return {"k": k, "v": v, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _materialize_own(s):
    k, v = _kvcache().materialize(_own_pool(s), s["tables"], s["starts"], first=s["past"], tokens=s["tokens"],
                                  dtype=DTYPES[s["case"]["dtype"]])
    return {"k": k, "v": v}


def _attention_own(s):
    case = s["case"]
    return _kvcache().attention(s["q"], _own_pool(s), s["tables"], s["lengths"], s["starts"], window=case["window"],
                                max_new=s["max_new"], max_length=s["max_length"], return_lse=case["lse"])


_run_own = {"plan": _plan_own, "append": _append_own, "materialize": _materialize_own, "attention": _attention_own}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------


def _exact_append(case, s, past, new):
    block, dim, kv = case["block"], case["dim"], case["kv"]
    tables = s["tables"].cpu().tolist()
    out = {}
    for side in ("k", "v"):
        codes, scales, x = s[side + "_codes"], s[side + "_scales"].double(), s[side].double()
        back, at = [], 0
        for r, (p, n) in enumerate(zip(past, new)):
            for column in range(p // block, _blocks(p + n, block)):
                low, high = max(p, column * block), min(p + n, (column + 1) * block)
                b, kept = tables[r][column], low - column * block
                mine = x[at + low - p: at + high - p].transpose(0, 1)  # [kv, tokens, dim]
                unit = mine.abs().amax((1, 2)) / 127
                old = codes[b, :, :kept].double()
                if kept:
                    was = scales[b]
                    now = torch.maximum(was, unit)
                    old = (old * (was / now)[:, None, None]).round()
                    unit = now
                scales[b] = unit
                fresh = (mine / unit.clamp(min=1e-300)[:, None, None]).round()
                back.append(torch.cat([old, fresh], 1) * unit[:, None, None])
            at += n
        out[side] = torch.cat(back, 1).transpose(0, 1).reshape(-1, kv, dim)
        out[side + "_scales"] = scales
    return out


def _exact_materialize(case, s, past, new):
    block, tables = case["block"], s["tables"]
    out = {}
    for side in ("k", "v"):
        rows = []
        for r, (p, n) in enumerate(zip(past, new)):
            ids = tables[r, : _blocks(p + n, block)].long()
            x = s[side + "_codes"][ids].double() * s[side + "_scales"][ids].double()[:, :, None, None]
            rows.append(x.transpose(1, 2).reshape(-1, case["kv"], case["dim"])[p: p + n])
        out[side] = torch.cat(rows)
    return out


def _exact_attention(case, s, past, new):
    block, kv, group, dim = case["block"], case["kv"], case["group"], case["dim"]
    outs, lses, at = [], [], 0
    for r, (p, n) in enumerate(zip(past, new)):
        ids = s["tables"][r, : _blocks(p + n, block)].long()
        k, v = (s[x + "_codes"][ids].double() * s[x + "_scales"][ids].double()[:, :, None, None] for x in ("k", "v"))
        k, v = (t.transpose(0, 1).reshape(kv, -1, dim)[:, : p + n] for t in (k, v))
        q = s["q"][at: at + n].double().view(n, kv, group, dim)
        at += n
        key, place = torch.arange(p + n, device=DEVICE), p + torch.arange(n, device=DEVICE)
        hidden = key[None] > place[:, None]
        if case["window"]:
            hidden |= key[None] + case["window"] <= place[:, None]
        out = torch.empty(n, kv, group, dim, dtype=torch.float64, device=DEVICE)
        lse = torch.empty(n, kv, group, dtype=torch.float64, device=DEVICE)
        for h in range(kv):
            for g in range(group):
                score = (q[:, h, g] @ k[h].T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                lse[:, h, g] = torch.logsumexp(score, 1)
                out[:, h, g] = torch.exp(score - lse[:, h, g, None]) @ v[h]
        outs.append(out.view(n, kv * group, dim))
        lses.append(lse.view(n, kv * group))
    out = torch.cat(outs)
    return (out, torch.cat(lses)) if case["lse"] else out


def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits; the whole numbers of a plan have no such value."""
    if case["op"] == "plan":
        return None
    form = {"append": _exact_append, "materialize": _exact_materialize, "attention": _exact_attention}[case["op"]]
    return form(case, prepare(case, seed), *_lengths(case))


def work(case):
    past, new = _lengths(case)
    block = case["block"]
    if case["op"] == "plan":
        tokens, gone = sum(max(n, 0) for n in new), sum(_blocks(p, block) for p, n in zip(past, new) if n < 0)
        fresh = sum(_blocks(p + max(n, 0), block) - _blocks(p, block) for p, n in zip(past, new))
        # two numbers read and two written a request, a slot and a position a token, each block that changes hands
        return {"bytes": 16 * len(past) + 12 * tokens + 8 * (fresh + gone) + 64, "flops": 0}
    row = 2 * case["kv"] * case["dim"]  # a token's keys and values
    scale = 2 * case["kv"] * 4 + 4      # a block's two scales of each head, and its place in the table
    tokens, held = sum(new), [p + n for p, n in zip(past, new)]
    if case["op"] == "append":
        touched = sum(_blocks(h, block) - p // block for h, p in zip(held, past))
        back = sum(h - p // block * block for h, p in zip(held, past))
        # 16 bits in, 8 out; what was touched read and written as 16 bits again
        return {"bytes": tokens * (3 * row + 8) + back * 3 * row + 2 * touched * scale, "flops": 2 * row * (tokens + back)}
    if case["op"] == "materialize":
        return {"bytes": tokens * 3 * row + sum(_blocks(h, block) for h in held) * scale, "flops": row * tokens}
    heads, window = case["kv"] * case["group"], case["window"] or 1 << 40
    # the keys that some query of the request sees, and all pairs of a query and a key that it sees
    keys = sum(h - max(0, p + 1 - window) for h, p in zip(held, past))
    pairs = sum(_pairs(p + n, window) - _pairs(p, window) for p, n in zip(past, new))
    return {"bytes": keys * (row + scale / block) + tokens * heads * (4 * case["dim"] + (4 if case["lse"] else 0)),
            "flops": 4 * pairs * heads * case["dim"]}


def _pairs(n, window):
    """Pairs of a query and a key that it sees, over the first n tokens of a request."""
    m = min(n, window)
    return m * (m + 1) // 2 + (n - m) * window
