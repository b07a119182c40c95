"""The 8-bit paged cache's kernels against the formulas in 64 bits.

Tolerances, fixed from the arithmetic:
* plan, and the codes and scales of append: equal bit for bit to 32-bit torch (the same IEEE
  operations in the same order).
* materialize: one rounding of code * scale, so equal to the rounded 32-bit product.
* attention: the products of codes are exact and sums are fp32; the weights of the values are
  rounded to fp16, an error of at most 2^-11 of each (and 2^-25 of the largest where they are
  subnormal), so an output is off by at most 2^-11 sum |w v| / l <= 2^-11 max |v| of its keys, plus
  its own rounding (2^-11 or 2^-8 of it).  The log-sum-exp is off by a few 2^-22 of the scores
  (fp32 products and sums, the approximate exponential and logarithm): 2^-17 (1 + max |score|).
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

kv = pytest.importorskip("mlbricks_b200.kvcache")


@pytest.fixture(autouse=True)
def _cuda(cuda_ok):
    torch.manual_seed(0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def blocks_of(n, b):
    return -(-n // b)


def make_tables(held, block, spare=2, width=None):
    """Shuffled blocks; entries that no token needs are garbage that must not be followed."""
    total = sum(blocks_of(h, block) for h in held)
    order = torch.randperm(total + spare).tolist()
    width = width or max(1, max(blocks_of(h, block) for h in held) + 1)
    tables = torch.randint(-(2**31), 2**31 - 1, (len(held), width), dtype=torch.int64).int()
    at = 0
    for i, h in enumerate(held):
        n = blocks_of(h, block)
        tables[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return tables.cuda(), total + spare


def make_pool(blocks, heads, block, dim, k_size=0.02, v_size=0.02):
    codes = [torch.randint(-127, 128, (blocks, heads, block, dim), dtype=torch.int8, device="cuda") for _ in "kv"]
    scales = [size * torch.exp(torch.randn(blocks, heads, device="cuda")) for size in (k_size, v_size)]
    return kv.KVPool(codes[0], scales[0], codes[1], scales[1])


def dense(pool, tables, i, n, side):
    """Request i's first n keys or values [n, heads, dim] in 64 bits."""
    b = pool.block_size
    ids = tables[i, :blocks_of(n, b)].long()
    codes, scales = (pool.k_codes, pool.k_scales) if side == "k" else (pool.v_codes, pool.v_scales)
    x = codes[ids].double() * scales[ids].double()[:, :, None, None]
    return x.transpose(1, 2).reshape(-1, pool.kv_heads, pool.head_dim)[:n]


def check_attention(q, pool, tables, lengths, new, out, lse, *, scale=None, causal=True, window=0, first=None):
    group = q.shape[1] // pool.kv_heads
    scale = 1 / math.sqrt(pool.head_dim) if scale is None else scale
    at = 0
    for i, (length, n) in enumerate(zip(lengths, new)):
        if n == 0:
            continue
        length = min(length, tables.shape[1] * pool.block_size)
        k, v = dense(pool, tables, i, length, "k"), dense(pool, tables, i, length, "v")
        p = length - n + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if causal:
            seen &= j <= p
        if window:
            seen &= j > p - window
        if first is not None:
            seen &= j >= first[i]
        empty = ~seen.any(1)
        for h in range(q.shape[1]):
            s = scale * (q[at:at + n, h].double() @ k[:, h // group].T)
            s = torch.where(seen, s, -math.inf)
            want_lse = torch.logsumexp(s, 1)
            w = torch.where(empty[:, None], 0.0, torch.exp(s - want_lse[:, None]))
            want = w @ v[:, h // group]
            got = out[at:at + n, h].double()
            assert torch.equal(got[empty], torch.zeros_like(got[empty]))
            size = (w @ v[:, h // group].abs()) + want.abs()
            eps = 2.0**-11 if q.dtype is torch.float16 else 2.0**-8
            tol = 2.0**-10 * size + 1.01 * eps * want.abs() + 2.0**-24
            assert torch.isfinite(got).all()
            assert ((got - want).abs() <= tol).all(), (i, h, ((got - want).abs() / tol).max())
            if lse is not None:
                g = lse[at:at + n, h].double()
                assert torch.equal(g[empty], torch.full_like(g[empty], -math.inf))
                top = torch.where(seen, s.abs(), 0.0).amax(1) if length else torch.zeros(n, device="cuda")
                assert ((g - want_lse).abs()[~empty] <= 2.0**-17 * (1 + top[~empty])).all()
        at += n


def run_attention(lengths, new, *, heads, group, dim, block, dtype=torch.float16, q_size=1.0, padded=0, **kw):
    tables, blocks = make_tables([max(x, 1) for x in lengths], block)
    pool = make_pool(blocks, heads, block, dim)
    tokens = sum(new)
    fused = q_size * torch.randn(tokens, heads * group + 3, dim, device="cuda")
    q = fused.to(dtype)[:, 1:1 + heads * group]
    starts = i32([sum(new[:i]) for i in range(len(new) + 1)])
    first = kw.pop("first", None)
    out, lse = kv.attention(q, pool, tables, i32(lengths), starts, return_lse=True,
                            first=None if first is None else i32(first), **kw)
    kw.pop("max_new", None), kw.pop("max_length", None)
    check_attention(q, pool, tables, lengths, new, out, lse, first=first, **kw)
    return q, pool, tables, starts, out, lse


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 640, 1000]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_single_tokens_of_every_length(block, dim, dtype):
    run_attention(LENGTHS, [1] * len(LENGTHS), heads=2, group=4, dim=dim, block=block, dtype=dtype, q_size=3.0)


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 12), (3, 5), (2, 16), (1, 17), (8, 1), (1, 40)])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_head_layouts(heads, group, dim):
    run_attention([77, 300, 5], [1, 3, 5], heads=heads, group=group, dim=dim, block=32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("block", [16, 64, 128])
def test_prompts_and_chunks(block, dim, dtype):
    run_attention([1, 130, 64, 333, 129, 700], [1, 130, 63, 200, 1, 129], heads=2, group=3, dim=dim, block=block,
                  dtype=dtype)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 7, 129, 300]])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 64, 100, 100000])
def test_windows(window, new):
    run_attention([500, 7, 129, 301], new, heads=2, group=4, dim=64, block=16, window=window)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 7, 129, 300]])
def test_without_causal_mask(new):
    run_attention([500, 7, 129, 301], new, heads=2, group=2, dim=128, block=64, causal=False)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.5])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 129, 300]])
def test_any_scale(new, scale):
    run_attention([500, 129, 301], new, heads=2, group=4, dim=64, block=16, scale=scale)
    run_attention([500, 129, 301], new, heads=1, group=5, dim=128, block=32, scale=scale, dtype=torch.bfloat16)


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [40, 7, 129, 300, 64]])
@pytest.mark.parametrize("window", [0, 33])
def test_first_leaves_rows_empty(new, window):
    # first past the length: nothing to see; in the middle of a prompt: its first rows see nothing
    run_attention([500, 7, 129, 301, 64], new, heads=2, group=4, dim=64, block=32, first=[3, 1000, 128, 150, 64],
                  window=window)


@pytest.mark.parametrize("new", [[1, 1], [40, 300]])
def test_numbers_as_large_as_they_go(new):
    most = 2**31 - 1
    run_attention([500, 200], new, heads=1, group=4, dim=64, block=32, first=[0, most], window=most)


def test_requests_without_tokens():
    run_attention([0, 5, 0, 9, 100, 0], [0, 5, 0, 1, 0, 0], heads=1, group=2, dim=32, block=16)


@pytest.mark.parametrize("group", [1, 4])
def test_more_queries_than_tokens_see_nothing(group):
    # a request that got no blocks: 3 queries over a cache of 1 token
    run_attention([1, 0, 20], [3, 2, 4], heads=2, group=group, dim=64, block=16)


@pytest.mark.parametrize("new", [1, 30, 70])
def test_hints_change_nothing(new):
    args = dict(heads=2, group=4, dim=128, block=16)
    outs = []
    for hints in ({}, {"max_new": new, "max_length": 900}, {"max_new": 1, "max_length": 1},
                  {"max_new": 5000, "max_length": 100000}):
        torch.manual_seed(3)
        outs.append(run_attention([900, 300], [new, new], **args, **hints)[4:])
    for out, lse in outs[1:]:
        assert (out.float() - outs[0][0].float()).abs().max() <= 2.0**-8 * outs[0][0].float().abs().max()


@pytest.mark.parametrize("new", [2, 3, 9])
def test_a_hint_that_is_too_small_leaves_no_row_out(new):
    run_attention([20011, 3000], [new, new], heads=2, group=4, dim=128, block=64, max_new=1)
    run_attention([20011, 3000], [new, new], heads=1, group=5, dim=32, block=16, max_new=1, max_length=9)


@pytest.mark.parametrize("dim,group,heads", [(128, 4, 2), (32, 12, 1), (64, 1, 3)])
@pytest.mark.parametrize("many", [3, 40])
def test_a_prompt_among_steps(many, dim, group, heads):
    """One prompt and `many` requests with a token or a few: both kernels, each for its own."""
    lengths = [20 + (331 * i) % 3000 for i in range(many)] + [400]
    new = [0 if i == 1 else 7 if i == 2 else 1 for i in range(many)] + [300]
    run_attention(lengths, new, heads=heads, group=group, dim=dim, block=32, max_new=300, max_length=3020)
    run_attention(lengths[::-1], new[::-1], heads=heads, group=group, dim=dim, block=32, max_new=300, window=70)


@pytest.mark.parametrize("requests", [1, 300])
def test_long_requests_are_split_and_joined(requests):
    lengths = [20011] if requests == 1 else [1 + (37 * i) % 900 for i in range(requests)]
    run_attention(lengths, [1] * requests, heads=2, group=4, dim=128, block=64, q_size=2.0)


@pytest.mark.parametrize("new", [1, 60])
def test_more_requests_than_a_window_of_the_shares(new):
    lengths = [new + (29 * i) % 90 for i in range(2100)]
    run_attention(lengths, [new if i % 3 == 0 or new == 1 else 0 for i in range(2100)], heads=1, group=1, dim=32, block=16)


def test_same_inputs_same_bits():
    q, pool, tables, starts, out, lse = run_attention([5000, 17, 900], [1, 1, 40], heads=4, group=4, dim=128, block=16)
    for _ in range(3):
        again = kv.attention(q, pool, tables, i32([5000, 17, 900]), starts, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_peaked_scores_and_scales_far_apart():
    """Scores of hundreds, V scales from 2^-90 to 2^15 in one row, and blocks of zeros."""
    tables, blocks = make_tables([600], 16)
    pool = make_pool(blocks, 1, 16, 64, k_size=0.05)
    pool.v_scales[:] = torch.exp2(torch.linspace(-90, 8, blocks, device="cuda"))[torch.randperm(blocks, device="cuda"), None]
    pool.v_scales[tables[0, 3].long()] = 0
    pool.v_codes[tables[0, 3].long()] = 0
    pool.k_scales[tables[0, 5].long()] = 0
    q = 8 * torch.randn(4, 6, 64, device="cuda", dtype=torch.float16)
    out, lse = kv.attention(q, pool, tables, i32([600]), i32([0, 4]), return_lse=True)
    check_attention(q, pool, tables, [600], [4], out, lse)


def test_bfloat16_queries_beyond_float16():
    tables, blocks = make_tables([300], 16)
    pool = make_pool(blocks, 2, 16, 64)
    q = (1e9 * torch.randn(3, 4, 64, device="cuda")).bfloat16()
    q[1] *= 2.0**-60
    out, lse = kv.attention(q, pool, tables, i32([300]), i32([0, 3]), scale=1e-9, return_lse=True)
    check_attention(q, pool, tables, [300], [3], out, lse, scale=1e-9)


@pytest.mark.parametrize("new", [1, 50])
def test_what_is_masked_is_never_seen(new):
    """NaN scales in blocks behind the window, before `first` and past the length, and in other requests."""
    length, block = 500, 16
    tables, blocks = make_tables([length, 40], block)
    pool = make_pool(blocks, 2, block, 64)
    args = dict(window=100, first=i32([430, 0]), return_lse=True)
    q = torch.randn(new, 4, 64, device="cuda", dtype=torch.float16)
    lengths, starts = i32([length, 40]), i32([0, new, new])
    clean = kv.attention(q, pool, tables, lengths, starts, **args)
    hidden = torch.ones(blocks, dtype=torch.bool, device="cuda")
    hidden[tables[0, 430 // block:blocks_of(length, block)].long()] = False
    for s in (pool.k_scales, pool.v_scales):
        s[hidden] = math.nan
    again = kv.attention(q, pool, tables, lengths, starts, **args)
    assert torch.equal(clean[0], again[0]) and torch.equal(clean[1], again[1])
    pool.v_scales[tables[0, length // block].long()] = math.nan  # and what is seen shows
    assert kv.attention(q, pool, tables, lengths, starts, **args)[0][-1].isnan().all()


def test_partly_masked_block_with_nan_scale_is_seen_only_where_it_is():
    """A NaN block that starts inside the window of some rows only."""
    tables, blocks = make_tables([64], 16)
    pool = make_pool(blocks, 1, 16, 32)
    pool.v_scales[tables[0, 3].long()] = math.nan
    q = torch.randn(64, 1, 32, device="cuda", dtype=torch.float16)
    out = kv.attention(q, pool, tables, i32([64]), i32([0, 64]))
    assert out[:48].isfinite().all() and out[48:].isnan().all()


def test_table_entries_out_of_range_are_not_seen():
    tables, blocks = make_tables([64, 64], 16)
    pool = make_pool(blocks, 1, 16, 64)
    q = torch.randn(2, 2, 64, device="cuda", dtype=torch.float16)
    want = kv.attention(q, pool, tables, i32([64, 64]), i32([0, 1, 2]), first=i32([0, 32]))
    tables[1, 0], tables[1, 1] = -1, blocks
    got = kv.attention(q, pool, tables, i32([64, 64]), i32([0, 1, 2]))
    assert (got.float() - want.float()).abs().max() < 1e-3


def test_pool_past_32_bit_offsets():
    """A block whose codes lie more than 2^32 bytes into the pool."""
    block, heads, dim = 128, 8, 128
    blocks = 2**32 // (block * heads * dim) + 40
    pool = kv.KVPool.empty(blocks, heads, block, dim)
    ids = [blocks - 1, 3, blocks - 7]
    tables = i32([ids])
    k = torch.randn(300, heads, dim, device="cuda", dtype=torch.float16)
    v = torch.randn(300, heads, dim, device="cuda", dtype=torch.float16)
    slots = torch.tensor([ids[p // block] * block + p % block for p in range(300)], device="cuda")
    kv.append(k, v, pool, slots)
    gk, gv = kv.materialize(pool, tables, i32([0, 300]), tokens=300, dtype=torch.float32)
    assert ((gk - k).abs().amax((0, 2)) <= k.abs().amax((0, 2)) / 250).all()
    assert ((gv - v).abs().amax((0, 2)) <= v.abs().amax((0, 2)) / 250).all()
    q = torch.randn(1, heads, dim, device="cuda", dtype=torch.float16)
    out, lse = kv.attention(q, pool, tables, i32([300]), i32([0, 1]), return_lse=True)
    check_attention(q, pool, tables, [300], [1], out, lse)


# ---- append and materialize -----------------------------------------------------------------


def append_reference(x, codes, scales, slots):
    """The formula, run by run, in the same 32-bit operations."""
    block = codes.shape[2]
    slots = slots.tolist()
    t = 0
    while t < len(slots):
        s = slots[t]
        if s < 0 or s >= codes.shape[0] * block:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == s + n and (s + n) % block:
            n += 1
        b, off = s // block, s % block
        mine = x[t:t + n].float().transpose(0, 1)  # [heads, n, dim]
        most = mine.abs().amax((1, 2))
        most = torch.where(most.isfinite(), most, math.nan)
        fresh = most / torch.full_like(most, 127.0)
        old = scales[b].clone() if off else torch.zeros_like(fresh)
        unit = torch.maximum(old, fresh)
        ratio = torch.where(unit > old, old / unit, 1.0)
        codes[b, :, :off] = (codes[b, :, :off].float() * ratio[:, None, None]).round().to(torch.int8)
        u = unit[:, None, None]
        codes[b, :, off:off + n] = torch.where(u > 0, mine / u, 0).round().clamp(-127, 127).to(torch.int8)
        scales[b] = unit
        t += n


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_equals_the_formula(block, dim, dtype):
    heads = 3
    past, new = [0, 5, 16, 31, 200, 0, 127], [1, 1, 33, 1, 150, 300, 2]
    tables, blocks = make_tables([p + n for p, n in zip(past, new)], block)
    pool = make_pool(blocks, heads, block, dim)
    want = [t.clone() for t in (pool.k_codes, pool.k_scales, pool.v_codes, pool.v_scales)]
    slots = [int(tables[i, p // block]) * block + p % block
             for i, (a, n) in enumerate(zip(past, new)) for p in range(a, a + n)]
    slots[34] = -1                       # a request's last token: its run ends ahead of it
    slots[185] = blocks * block + 5      # past the pool
    slots = torch.tensor(slots, device="cuda")
    fused = torch.randn(len(slots), 2 * heads + 1, dim, device="cuda").to(dtype) * 4
    k, v = fused[:, 1:1 + heads], fused[:, 1 + heads:]
    k[3] = 0
    kv.append(k, v, pool, slots)
    append_reference(k, want[0], want[1], slots)
    append_reference(v, want[2], want[3], slots)
    for got, w in zip((pool.k_codes, pool.k_scales, pool.v_codes, pool.v_scales), want):
        assert torch.equal(got, w)
    again = [t.clone() for t in (pool.k_codes, pool.v_codes)]
    kv.append(k, v, pool, slots)  # the same tokens once more change nothing
    assert torch.equal(pool.k_codes, again[0]) and torch.equal(pool.v_codes, again[1])


def test_append_many_tokens_by_the_longer_span():
    block, heads, dim = 64, 4, 64
    past, new = [3, 0, 700], [2500, 1, 1900]
    tables, blocks = make_tables([p + n for p, n in zip(past, new)], block)
    pool = make_pool(blocks, heads, block, dim)
    want = [t.clone() for t in (pool.k_codes, pool.k_scales)]
    slots = torch.cat([tables[i, torch.arange(p, p + n) // block].long() * block + torch.arange(p, p + n, device="cuda") % block
                       for i, (p, n) in enumerate(zip(past, new))])
    k = torch.randn(len(slots), heads, dim, device="cuda", dtype=torch.float16)
    kv.append(k, k, pool, slots)
    append_reference(k, want[0], want[1], slots)
    assert torch.equal(pool.k_codes, want[0]) and torch.equal(pool.k_scales, want[1])


def test_append_zeros_ties_and_non_finite_values():
    pool = kv.KVPool.empty(5, 1, 16, 32)
    k = torch.zeros(40, 1, 32, device="cuda", dtype=torch.float16)
    k[16:32] = torch.arange(-254, 258, 1, device="cuda").view(16, 1, 32).clamp(-254, 254).half() / 2  # ties: n + 1/2
    k[33, 0, 3] = math.inf
    v = torch.zeros_like(k)
    v[5, 0, 0] = math.nan
    kv.append(k, v, pool, torch.arange(40, device="cuda"))
    assert pool.k_scales[0, 0] == 0 and not pool.k_codes[0].any()
    assert pool.k_scales[1, 0] == 1
    assert torch.equal(pool.k_codes[1].float(), k[16:32].float().transpose(0, 1).round())
    assert pool.k_scales[2, 0].isnan() and pool.v_scales[0, 0].isnan() and pool.v_scales[1, 0] == 0
    # a NaN block stays NaN when more tokens come
    kv.append(k[:1], v[:1], pool, torch.tensor([40], device="cuda"))
    assert pool.k_scales[2, 0].isnan()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads", [(32, 1), (64, 3), (128, 2)])
def test_materialize_rounds_once(dim, heads, dtype):
    held = [40, 1, 0, 129]
    tables, blocks = make_tables([max(h, 1) for h in held], 32)
    pool = make_pool(blocks, heads, 32, dim)
    first, counts = [3, 0, 0, 100], [37, 1, 0, 29]
    starts = i32([sum(counts[:i]) for i in range(5)])
    tokens = sum(counts) + 3  # rows of no request are 0
    got = kv.materialize(pool, tables, starts, first=i32(first), tokens=tokens, dtype=dtype)
    for side, x in zip("kv", got):
        codes, scales = (pool.k_codes, pool.k_scales) if side == "k" else (pool.v_codes, pool.v_scales)
        at = 0
        for i, (f, n) in enumerate(zip(first, counts)):
            p = torch.arange(f, f + n, device="cuda")
            ids = tables[i, p // 32].long()
            want = (codes[ids, :, p % 32].float() * scales[ids][:, :, None]).to(dtype)
            assert torch.equal(x[at:at + n], want)
            at += n
        assert not x[at:].any()


# ---- plan -----------------------------------------------------------------------------------


def plan_reference(past, new, tables, free, ring, block):
    """Request by request, on the host."""
    head, tail, size = ring[0], ring[1], len(free)
    avail, taken, gone, short = tail - head, 0, 0, 0
    lengths, starts, slots, positions = [], [0], [], []
    tables, free = [list(r) for r in tables], list(free)
    before = 0
    for i, (p, n) in enumerate(zip(past, new)):
        if n < 0:
            for j in range(blocks_of(p, block)):
                free[(tail + gone) % size] = tables[i][j]
                gone += 1
            lengths.append(0)
            starts.append(starts[-1])
            continue
        had, all_ = blocks_of(p, block), blocks_of(p + n, block)
        need = all_ - had
        fits = all_ <= len(tables[i]) and (need == 0 or before + need <= avail)
        if all_ <= len(tables[i]):
            if fits:
                for j in range(need):
                    tables[i][had + j] = free[(head + before + j) % size]
                taken = max(taken, before + need) if need else taken
            before += need
        if not fits:
            short += need
        lengths.append(p + n if fits else p)
        starts.append(starts[-1] + n)
        for x in range(p, p + n):
            positions.append(x)
            slots.append(tables[i][x // block] * block + x % block if fits else -1)
    return lengths, starts, slots, positions, [head + taken, tail + gone, short, starts[-1]], tables, free


@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("requests,most,spare", [(1, 500, 40), (7, 60, 3), (300, 40, 1000), (700, 100, 100), (3, 9000, 2000)])
def test_plan_equals_the_host(requests, most, spare, block):
    g = torch.Generator().manual_seed(requests + block)
    past = torch.randint(0, most, (requests,), generator=g).tolist()
    new = [x - 1 if x < 30 else x for x in torch.randint(0, 30 + most // 4, (requests,), generator=g).tolist()]
    held = sum(blocks_of(p, block) for p in past)
    width = blocks_of(most, block) + 1
    order = torch.randperm(held + spare, generator=g).tolist()
    tables = [[-1] * width for _ in past]
    at = 0
    for i, p in enumerate(past):
        for j in range(blocks_of(p, block)):
            tables[i][j] = order[at]
            at += 1
    size = held + spare
    head = 10**10 + 17  # far past 32 bits
    free = [0] * size
    for j in range(spare):
        free[(head + j) % size] = order[held + j]
    ring = [head, head + spare]
    tokens = sum(max(n, 0) for n in new) + 5
    d_tables, d_free = i32(tables), i32(free)
    step = kv.plan(i32(past), i32(new), d_tables, d_free, torch.tensor(ring, device="cuda"), block_size=block, tokens=tokens)
    lengths, starts, slots, positions, out, tables, free = plan_reference(past, new, tables, free, ring, block)
    assert step.ring.tolist() == out
    assert step.lengths.tolist() == lengths and step.starts.tolist() == starts
    assert step.slots.tolist() == slots + [-1] * 5 and step.positions.tolist() == positions + [0] * 5
    assert d_tables.tolist() == tables and d_free.tolist() == free


def test_plan_with_no_requests_and_no_tokens():
    step = kv.plan(i32([]), i32([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), i32([1, 2]),
                   torch.tensor([0, 2], device="cuda"), block_size=16, tokens=0)
    assert step.starts.tolist() == [0] and step.ring.tolist() == [0, 2, 0, 0]
    step = kv.plan(i32([16]), i32([0]), i32([[1]]), i32([1, 2]), torch.tensor([0, 1], device="cuda"), block_size=16, tokens=0)
    assert step.lengths.tolist() == [16]


def test_plan_with_numbers_out_of_range():
    """Lengths that no table holds, a ring that ends ahead of its front: nobody gets a block, nothing is followed."""
    most = 2**31 - 1
    tables, free = i32([[0, 1], [2, 3], [4, 5]]), i32([6, 7, 8])
    step = kv.plan(i32([most, -3, 40]), i32([5, 4, -1]), tables, free, torch.tensor([-9, -20], device="cuda"),
                   block_size=16, tokens=9)
    assert step.lengths.tolist() == [most, 0, 0] and step.slots.tolist() == [-1] * 9
    assert step.ring.tolist()[:2] == [0, 2]  # the third's two blocks (its row holds no more) join the ring
    assert free.tolist() == [4, 5, 8] and tables.tolist() == [[0, 1], [2, 3], [4, 5]]


# ---- refusals and streams -------------------------------------------------------------------


def test_refusals():
    pool = kv.KVPool.empty(4, 2, 16, 64)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.float16)
    ok = dict(tables=i32([[0]]), lengths=i32([1]), starts=i32([0, 1]))
    kv.attention(q, pool, **ok)
    bad = [
        (lambda: kv.KVPool.empty(4, 2, 24, 64), "block_size"),
        (lambda: kv.KVPool.empty(4, 2, 16, 96), "head_dim"),
        (lambda: kv.KVPool(pool.k_codes, pool.k_scales[:2], pool.v_codes, pool.v_scales), "k_scales"),
        (lambda: kv.KVPool(pool.k_codes.cpu(), pool.k_scales, pool.v_codes, pool.v_scales), "CUDA"),
        (lambda: kv.attention(q.float(), pool, **ok), "float16 or bfloat16"),
        (lambda: kv.attention(q[:, :3], pool, **ok), "multiple of kv_heads"),
        (lambda: kv.attention(q[..., :32], pool, **ok), "head"),
        (lambda: kv.attention(q, pool, **{**ok, "lengths": i32([1, 2])}), "as many"),
        (lambda: kv.attention(q, pool, **{**ok, "lengths": torch.ones(1, device="cuda", dtype=torch.int64)}), "lengths"),
        (lambda: kv.attention(q, pool, **ok, first=i32([1, 2])), "first"),
        (lambda: kv.attention(q, pool, **ok, window=-1), "window"),
        (lambda: kv.attention(q, pool, **ok, window=4, causal=False), "window"),
        (lambda: kv.attention(q, pool, **ok, scale=math.inf), "scale"),
        (lambda: kv.attention(q, pool, **ok, out=q.float()), "out"),
        (lambda: kv.append(q, q, pool, torch.zeros(1, dtype=torch.int64, device="cuda")), "tokens, 2"),
        (lambda: kv.append(q[:, :2], q[:, :2].bfloat16(), pool, torch.zeros(1, dtype=torch.int64, device="cuda")), "same"),
        (lambda: kv.append(q[:, :2], q[:, :2], pool, i32([0])), "slots"),
        (lambda: kv.materialize(pool, i32([[0]]), i32([0, 1]), tokens=1, dtype=torch.float64), "dtype"),
        (lambda: kv.materialize(pool, i32([[0]]), i32([0]), tokens=1), "row"),
        (lambda: kv.plan(i32([1]), i32([1, 2]), i32([[0]]), i32([1]), torch.tensor([0, 1], device="cuda"), block_size=16, tokens=1), "as many"),
        (lambda: kv.plan(i32([1]), i32([1]), i32([[0]]), i32([1]), torch.tensor([0, 1], device="cuda"), block_size=20, tokens=1), "block_size"),
        (lambda: kv.plan(i32([1]), i32([1]), i32([[0]]), i32([1]), i32([0, 1]), block_size=16, tokens=1), "ring"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()


def test_unaligned_and_strided_rows():
    tables, blocks = make_tables([50], 16)
    pool = make_pool(blocks, 2, 16, 64)
    base = torch.randn(3 * 4 * 64 + 3, device="cuda", dtype=torch.float16)
    q = base[3:].view(3, 4, 64)  # 6 bytes off
    args = (pool, tables, i32([50]), i32([0, 3]))
    want = kv.attention(q.clone(), *args)
    assert torch.equal(kv.attention(q, *args), want)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(kv.attention(turned, *args), want)
    spread = torch.stack([q, q], -1)[..., 0]
    assert torch.equal(kv.attention(spread, *args), want)


def test_other_streams_and_graphs():
    tables, blocks = make_tables([3000, 40], 64)
    pool = make_pool(blocks, 2, 64, 128)
    q = torch.randn(2, 8, 128, device="cuda", dtype=torch.float16)
    args = (q, pool, tables, i32([3000, 40]), i32([0, 1, 2]))
    want = kv.attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv.attention(*args)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.graph(graph):
        captured = kv.attention(*args)
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(captured, kv.attention(*args))


def test_device_status_is_clean():
    import ctypes

    from mlbricks_b200 import _ebx

    st = ctypes.c_int32(7)
    _ebx.check(_ebx.load().ebx_device_status(0, ctypes.byref(st), 0))
    assert st.value == 0
