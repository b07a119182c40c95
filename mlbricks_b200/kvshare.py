"""Requests that share blocks of the 8-bit paged key/value cache (``libebx``, include/ebx.h ``ebx_kv_*``).

Samples of one prompt, beams, and conversations behind one system prompt hold the same first tokens.  Here
they hold the same blocks, each with a count of its holders:

* ``fork``       lets rows go on from what other rows hold, rolls rows back, and frees them;
* ``compact``    moves the blocks that rows hold to the front of the pool;
* ``copy``       copies the blocks that either asks for, in all layers;
* ``prefixes``   finds which of a step's requests share a prefix;
* ``attention``  attends over the cache, reading what requests share once for all of them.

``SharedKVCache`` is a ``KVCache`` with all of them.

Inference only: no autograd.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Sequence

import torch

from . import _ebx
from .kvcache import _ROW_DTYPES, BLOCK_SIZES, KVCache, KVPlan, KVPool, _int_ok, _refuse_ints, _stream


MOST_REQUESTS = 8192  # of a step whose prefixes are looked for


class KVMoves(NamedTuple):
    """Blocks to copy (on the GPU)."""

    sources: torch.Tensor  # int32, -1 behind the last copy
    targets: torch.Tensor  # int32, likewise
    count: torch.Tensor    # int64 [1]


class KVFork(NamedTuple):
    """What ``fork`` wrote (all on the GPU)."""

    lengths: torch.Tensor  # int32 [requests]
    tables: torch.Tensor   # int32 [requests, width], -1 behind what a row holds
    shares: torch.Tensor   # int32 [blocks], holders beyond the first
    ring: torch.Tensor     # int64 [4]: front, back, blocks that were missing, copies
    moves: KVMoves


class KVCompact(NamedTuple):
    """What ``compact`` wrote (all on the GPU)."""

    tables: torch.Tensor   # int32 [requests, width]
    shares: torch.Tensor   # int32 [blocks]
    free: torch.Tensor     # int32 [blocks], the free blocks' numbers, then -1
    ring: torch.Tensor     # int64 [4]: 0, free blocks, 0, copies
    moves: KVMoves


def _state(lengths, tables, shares, block_size, device) -> None:
    """What fork and compact have in common."""
    int32 = torch.int32
    if device < 0:
        raise ValueError("lengths must be a CUDA tensor")
    if not (_int_ok(lengths, int32, device) and _int_ok(tables, int32, device) and _int_ok(shares, int32, device)):
        _refuse_ints(device, lengths=(lengths, int32), tables=(tables, int32), shares=(shares, int32))
    if tables.dim() != 2 or lengths.numel() != tables.shape[0] or tables.shape[1] < 1:
        raise ValueError("tables must have a row for each of lengths, and a column")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    if shares.numel() < 1:
        raise ValueError("shares must have an entry for each block")


def fork(lengths: torch.Tensor, tables: torch.Tensor, shares: torch.Tensor, free: torch.Tensor, ring: torch.Tensor,
         parents: torch.Tensor, *, block_size: int, keep: torch.Tensor | None = None) -> KVFork:
    """Rows of a block table that go on from others, in one launch.

    Row i continues the first ``keep[i]`` tokens (default, and at most: all) of what row ``parents[i]``
    (int32) held: its own number leaves it as it is or rolls it back, another row's forks that one, and a number that is no row
    (-1) frees the row.  All rows change at once, so beams may change places.  Full blocks are
    shared and counted in ``shares`` (int32, an entry for each block: holders beyond the first).  A block that is
    begun stays with one row; the others get a block each from the ring's front in row order, to be filled by ``copy`` with
    the result's ``moves``.  A row for which there is none is empty afterwards (length 0), and ``ring[2]`` of the result
    counts it.  Blocks without a holder join the ring's back (written in place in ``free``), by rising number, for
    later calls.

    ``lengths``, ``tables``, ``shares`` and ``ring`` are not changed: the result's take their place."""
    int32, device = torch.int32, lengths.get_device()
    _state(lengths, tables, shares, block_size, device)
    if not (_int_ok(free, int32, device) and _int_ok(ring, torch.int64, device) and _int_ok(parents, int32, device)
            and (keep is None or _int_ok(keep, int32, device))):
        _refuse_ints(device, free=(free, int32), ring=(ring, torch.int64), parents=(parents, int32), keep=(keep, int32))
    requests, width = tables.shape
    if parents.numel() != requests or (keep is not None and keep.numel() != requests):
        raise ValueError("parents and keep must have one entry for each request")
    if ring.numel() < 2 or free.numel() < 1:
        raise ValueError("ring holds at least its front and back, and free at least one place")
    blocks = shares.numel()
    # one allocation: cheaper than five
    cells = requests * width
    out_lengths, sources, targets, out_shares, out_tables = lengths.new_empty(3 * requests + blocks + cells).split_with_sizes(
        (requests, requests, requests, blocks, cells))
    out_tables, out_ring = out_tables.view(requests, width), ring.new_empty(4)
    st = _ebx.load().ebx_kv_fork(
        lengths.data_ptr(), tables.data_ptr(), width, block_size, shares.data_ptr(), blocks, free.data_ptr(), free.numel(),
        ring.data_ptr(), parents.data_ptr(), None if keep is None else keep.data_ptr(), requests, out_lengths.data_ptr(),
        out_tables.data_ptr(), out_shares.data_ptr(), out_ring.data_ptr(), sources.data_ptr(), targets.data_ptr(), device,
        _stream(device))
    if st:
        _ebx.check(st)
    return KVFork(out_lengths, out_tables, out_shares, out_ring, KVMoves(sources, targets, out_ring[3:]))


def compact(lengths: torch.Tensor, tables: torch.Tensor, shares: torch.Tensor, *, block_size: int) -> KVCompact:
    """New numbers for the blocks that rows hold, so that they are the pool's first ones, with the fewest copies
    (the result's ``moves``, for ``copy``).  All others are free afterwards, and in the result's ring by rising number.
    The inputs are not changed: the result's tensors take their place.  At most 524288 blocks."""
    device = lengths.get_device()
    _state(lengths, tables, shares, block_size, device)
    requests, width = tables.shape
    blocks = shares.numel()
    cells, half = requests * width, blocks // 2
    out_shares, free, sources, targets, out_tables = lengths.new_empty(2 * blocks + 2 * half + cells).split_with_sizes(
        (blocks, blocks, half, half, cells))
    out_tables, ring = out_tables.view(requests, width), lengths.new_empty(4, dtype=torch.int64)
    st = _ebx.load().ebx_kv_compact(
        lengths.data_ptr(), tables.data_ptr(), width, block_size, shares.data_ptr(), blocks, requests, out_tables.data_ptr(),
        out_shares.data_ptr(), free.data_ptr(), ring.data_ptr(), sources.data_ptr(), targets.data_ptr(), device,
        _stream(device))
    if st:
        _ebx.check(st)
    return KVCompact(out_tables, out_shares, free, ring, KVMoves(sources, targets, ring[3:]))


def copy(pools: Sequence[KVPool], moves: KVMoves) -> None:
    """Blocks ``moves.sources`` to ``moves.targets``, codes and scales, in every pool (layers of equal sizes), in place.
    Pairs with a number that is no block are skipped; no target is another pair's source or target."""
    if not pools:
        return
    device = pools[0].device
    sources, targets, count = moves
    if not (_int_ok(sources, torch.int32, device) and _int_ok(targets, torch.int32, device)
            and (count is None or _int_ok(count, torch.int64, device))):
        _refuse_ints(device, sources=(sources, torch.int32), targets=(targets, torch.int32), count=(count, torch.int64))
    if sources.numel() != targets.numel() or (count is not None and count.numel() < 1):
        raise ValueError("sources and targets must be as many, and count one number")
    array = (_ebx.KVPool * len(pools))(*[p._c for p in pools])
    st = _ebx.load().ebx_kv_copy(array, len(pools), sources.data_ptr(), targets.data_ptr(),
                                 None if count is None else count.data_ptr(), sources.numel(), _stream(device))
    if st:
        _ebx.check(st)


class KVPrefixes:
    """Which requests of a step share a prefix (``prefixes``)."""

    __slots__ = ("data", "requests", "tokens")

    def __init__(self, data: torch.Tensor, requests: int, tokens: int) -> None:
        self.data, self.requests, self.tokens = data, requests, tokens


def prefixes(tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, *, block_size: int, blocks: int,
             tokens: int) -> KVPrefixes:
    """Which requests of a step share a prefix, for ``attention`` of every layer.

    ``lengths`` and ``starts`` are the step's, as for ``kvcache.attention``; ``blocks`` is the pool's.  Requests that
    bring tokens and whose rows of ``tables`` begin with the same block form a group, which shares as many full blocks ahead
    of the new tokens as save most reading; rows with fewer in common are taken alone.  The result holds for this
    step.  At most 8192 requests."""
    int32, device, requests = torch.int32, tables.get_device(), lengths.numel()
    if device < 0:
        raise ValueError("tables must be a CUDA tensor")
    if not (_int_ok(tables, int32, device) and _int_ok(lengths, int32, device) and _int_ok(starts, int32, device)):
        _refuse_ints(device, tables=(tables, int32), lengths=(lengths, int32), starts=(starts, int32))
    if starts.numel() != requests + 1 or tables.dim() != 2 or tables.shape[0] != requests or tokens < 0:
        raise ValueError("lengths and the rows of tables must be as many, and starts one more; tokens >= 0")
    data = starts.new_empty(3 * requests + 2 + 2 * tokens)
    st = _ebx.load().ebx_kv_prefixes(tables.data_ptr(), tables.shape[1], block_size, blocks, lengths.data_ptr(), starts.data_ptr(),
                                     requests, tokens, data.data_ptr(), device, _stream(device))
    if st:
        _ebx.check(st)
    return KVPrefixes(data, requests, tokens)


@functools.lru_cache(maxsize=1024)
def _workspace(device: int, kv_heads: int, head_dim: int, heads: int, requests: int, tokens: int, max_new: int,
               max_length: int) -> tuple[int, bool]:
    """Bytes of workspace, and whether prefixes are used at all."""
    pool = ctypes.byref(_ebx.KVPool(16, 16, 16, 16, 1, kv_heads, BLOCK_SIZES[0], head_dim, device, 0))  # only its sizes count
    sizes, lib = (heads, requests, tokens, max_new, max_length), _ebx.load()
    return int(lib.ebx_kv_shared_attention_workspace_bytes(pool, *sizes)), bool(lib.ebx_kv_takes_prefixes(pool, *sizes))


def takes_prefixes(pool: KVPool, heads: int, requests: int, tokens: int, max_new: int = 0, max_length: int = 0) -> bool:
    """Whether ``attention`` with these sizes uses prefixes; where it does not, ``prefixes`` need not be called."""
    if heads <= 0 or heads % pool.kv_heads or min(requests, tokens, max_new, max_length) < 0 or requests > MOST_REQUESTS:
        return False
    return _workspace(pool.device, pool.kv_heads, pool.head_dim, heads, requests, tokens, max_new, max_length)[1]


def attention(q: torch.Tensor, pool: KVPool, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
              shared: KVPrefixes, *, scale: float | None = None, causal: bool = True, max_new: int = 0, max_length: int = 0,
              out: torch.Tensor | None = None, return_lse: bool = False):
    """``kvcache.attention`` (without ``window`` and ``first``) that reads the prefixes that ``shared`` tells of, found
    by ``prefixes`` for the same tables, lengths and starts, once for all requests that share them.

    The formula is the same; the order of sums is not.  ``out``, if given, is not q's memory.  ``max_new``, the largest
    number of new tokens of a request, should be given: with 49 rows (max_new, or without it tokens, times heads /
    kv_heads) and more, all requests go by themselves; so they do where requests and ``max_length``, if given, are too
    few for sharing to pay (``takes_prefixes``).  ``max_length`` decides best as the largest length that there is, not
    one that there may be."""
    q = pool._rows(q, None, "q")
    device, int32 = pool.device, torch.int32
    tokens, heads, dim = q.shape
    requests = lengths.numel()
    if not (_int_ok(tables, int32, device) and _int_ok(lengths, int32, device) and _int_ok(starts, int32, device)
            and _int_ok(shared.data, int32, device)):
        _refuse_ints(device, tables=(tables, int32), lengths=(lengths, int32), starts=(starts, int32), shared=(shared.data, int32))
    if heads == 0 or heads % pool._c.kv_heads:
        raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({pool._c.kv_heads})")
    if starts.numel() != requests + 1 or tables.dim() != 2 or tables.shape[0] != requests:
        raise ValueError("lengths and the rows of tables must be as many, and starts one more")
    if shared.requests != requests or shared.tokens != tokens or shared.data.numel() != 3 * requests + 2 + 2 * tokens:
        raise ValueError("shared must be of this step: as many requests and tokens")
    if out is None:
        out = torch.empty_like(q)  # cheaper than new_empty, and contiguous unless q is dense in another order
        if not out.is_contiguous():
            out = q.new_empty((tokens, heads, dim))
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != device or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape and dtype")
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    if tokens and requests:
        nbytes = _workspace(device, pool._c.kv_heads, dim, heads, requests, tokens, max_new, max_length)[0]
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        st = _ebx.load().ebx_kv_shared_attention(
            pool._ref, q.data_ptr(), q.stride(0), q.stride(1), heads, _ROW_DTYPES[q.dtype], tables.data_ptr(),
            tables.shape[1], lengths.data_ptr(), starts.data_ptr(), shared.data.data_ptr(), requests, tokens, causal,
            1.0 / math.sqrt(dim) if scale is None else scale, max_new, max_length, out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, _stream(device))
        if st:
            _ebx.check(st)
    return out if lse is None else (out, lse)


class SharedKVCache(KVCache):
    """A ``KVCache`` whose requests can share blocks.

    ``fork`` makes rows go on from others, frees them and rolls them back, ``compact`` renumbers blocks; both
    come between steps: a step is planned after them.  ``attention`` reads prefixes that requests share once, where
    ``takes_prefixes`` says that it pays if requests are as long as ``max_length``: a cache much larger than what it holds
    is better a ``KVCache`` if nothing is shared."""

    def __init__(self, layers: int, blocks: int, kv_heads: int, head_dim: int, *, requests: int, max_length: int,
                 block_size: int = 64, device="cuda") -> None:
        super().__init__(layers, blocks, kv_heads, head_dim, requests=requests, max_length=max_length,
                         block_size=block_size, device=device)
        where = self.lengths.device
        self.shares = torch.zeros(blocks, dtype=torch.int32, device=where)
        self._rows = torch.arange(requests, dtype=torch.int32, device=where)
        self._shared: KVPrefixes | None = None

    def plan(self, new, tokens: int | None = None, max_new: int | None = None, releases: bool = True) -> KVPlan:
        """As ``KVCache.plan``, but a request that is done (-1) gives up blocks that it shares, and its blocks are there
        for this step already.  With a tensor ``new`` that costs a launch or two more, unless ``releases`` is False:
        then -1 is taken for 0."""
        # all that can be refused is, before a row is freed
        requests, where = self._rows.numel(), self.lengths.device
        listed = not isinstance(new, torch.Tensor)
        if listed:
            new = [int(n) for n in new]
            done = [-1 if n < 0 else i for i, n in enumerate(new)] if min(new, default=0) < 0 else None
            counts = [max(n, 0) for n in new]
            tokens, max_new = sum(counts), max(counts, default=0)
            new = torch.tensor(counts, dtype=torch.int32).to(where, non_blocking=True)
        elif not _int_ok(new, torch.int32, self.lengths.get_device()):
            _refuse_ints(self.lengths.get_device(), new=(new, torch.int32))
        if new.numel() != requests:
            raise ValueError(f"new must have an entry for each of the {requests} requests")
        if tokens is None or not 0 <= tokens < 2**31:
            raise ValueError("a tensor of new tokens needs `tokens`, 0 <= tokens < 2^31")
        if not listed:
            new = new.view(-1)
            if releases:
                self.fork(torch.where(new < 0, -1, self._rows).to(torch.int32))
            new = new.clamp(min=0)
        elif done is not None:
            self.fork(done)
        self._shared = None
        return super().plan(new, tokens, max_new)

    def fork(self, parents, keep=None) -> KVFork:
        """Row i goes on from the first ``keep[i]`` tokens (default: all) of row ``parents[i]``; -1 frees it.  Lists, or
        int32 tensors on the GPU.  Returns ``fork``'s result, whose copies are made; ``ring[2]`` counts rows that found no block
        and are empty now."""
        parents, keep = (x if x is None or isinstance(x, torch.Tensor) else
                         torch.tensor([int(n) for n in x], dtype=torch.int32).to(self.lengths.device, non_blocking=True)
                         for x in (parents, keep))
        done = fork(self.lengths, self.tables, self.shares, self.free, self.ring, parents, block_size=self.block_size, keep=keep)
        copy(self.pools, done.moves)
        self.lengths.copy_(done.lengths)
        self._take(done)
        return done

    def compact(self) -> KVCompact:
        """Moves the blocks that rows hold to the front of the pools.  Returns ``compact``'s result, whose copies are made."""
        done = compact(self.lengths, self.tables, self.shares, block_size=self.block_size)
        copy(self.pools, done.moves)
        self.free.copy_(done.free)
        self._take(done)
        return done

    def _take(self, done: KVFork | KVCompact) -> None:
        self.tables.copy_(done.tables)
        self.shares.copy_(done.shares)
        self.ring.copy_(done.ring)
        self.step = self._shared = None  # slots and prefixes of a step planned before are not this table's

    def attention(self, layer: int, q: torch.Tensor, **options):
        """The step's queries over the layer's cache, what requests share once; as ``KVCache.attention`` with ``window`` or
        ``first``, which prefixes do not allow, and where sharing could not pay."""
        step = self._planned()
        if (options.get("window") or options.get("first") is not None or q.dim() != 3
                or not takes_prefixes(self.pools[layer], q.shape[1], self.lengths.numel(), q.shape[0], self._max_new,
                                      self.max_length)):
            return super().attention(layer, q, **options)
        options.pop("window", None), options.pop("first", None)
        if self._shared is None or self._shared.tokens != q.shape[0]:  # a layer may bring fewer queries
            self._shared = prefixes(self.tables, step.lengths, step.starts, block_size=self.block_size,
                                    blocks=self.pools[layer].blocks, tokens=q.shape[0])
        return attention(q, self.pools[layer], self.tables, step.lengths, step.starts, self._shared,
                         max_new=self._max_new, max_length=self.max_length, **options)


__all__ = ["KVCompact", "KVFork", "KVMoves", "KVPrefixes", "SharedKVCache", "attention", "compact", "copy", "fork", "prefixes",
           "takes_prefixes"]
