"""Requests that share blocks of the 8-bit paged key/value cache (``libebx``, include/ebx.h ``ebx_kv_*``).

Samples of one prompt, beams, and conversations behind one system prompt hold the same first tokens.  Here
they hold the same blocks, each with a count of its holders:

* ``fork``       lets rows go on from what other rows hold, rolls rows back, and frees them;
* ``compact``    moves the blocks that rows hold to the front of the pool;
* ``copy``       copies the blocks that either asks for, in all layers;

Inference only: no autograd.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from . import _ebx
from .kvcache import BLOCK_SIZES, KVPool, _int_ok, _refuse_ints, _stream


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


def _state(lengths: torch.Tensor, tables: torch.Tensor, shares: torch.Tensor, block_size: int, **more) -> int:
    """Checks what fork and compact have in common; the device."""
    device = lengths.get_device()
    if device < 0:
        raise ValueError("lengths must be a CUDA tensor")
    int32 = torch.int32
    _refuse_ints(device, lengths=(lengths, int32), tables=(tables, int32), shares=(shares, int32), **more)
    if tables.dim() != 2 or lengths.numel() != tables.shape[0] or tables.shape[1] < 1:
        raise ValueError("tables must have a row for each of lengths, and a column")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    if shares.numel() < 1:
        raise ValueError("shares must have an entry for each block")
    return device


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
    int32 = torch.int32
    device = _state(lengths, tables, shares, block_size, free=(free, int32), ring=(ring, torch.int64),
                    parents=(parents, int32), keep=(keep, int32))
    requests, width = tables.shape
    if parents.numel() != requests or (keep is not None and keep.numel() != requests):
        raise ValueError("parents and keep must have one entry for each request")
    if ring.numel() < 2 or free.numel() < 1:
        raise ValueError("ring holds at least its front and back, and free at least one place")
    blocks = shares.numel()
    out_lengths, out_tables, out_shares = lengths.new_empty(requests), tables.new_empty((requests, width)), shares.new_empty(blocks)
    out_ring, moves, work = ring.new_empty(4), lengths.new_empty((2, requests)), shares.new_empty(blocks)
    _ebx.check(_ebx.load().ebx_kv_fork(
        lengths.data_ptr(), tables.data_ptr(), width, block_size, shares.data_ptr(), blocks, free.data_ptr(), free.numel(),
        ring.data_ptr(), parents.data_ptr(), None if keep is None else keep.data_ptr(), requests, out_lengths.data_ptr(),
        out_tables.data_ptr(), out_shares.data_ptr(), out_ring.data_ptr(), moves[0].data_ptr(), moves[1].data_ptr(),
        work.data_ptr(), 4 * blocks, device, _stream(device)))
    return KVFork(out_lengths, out_tables, out_shares, out_ring, KVMoves(moves[0], moves[1], out_ring[3:]))


def compact(lengths: torch.Tensor, tables: torch.Tensor, shares: torch.Tensor, *, block_size: int) -> KVCompact:
    """New numbers for the blocks that rows hold, so that they are the pool's first ones, with the fewest copies
    (the result's ``moves``, for ``copy``).  All others are free afterwards, and in the result's ring by rising number.
    The inputs are not changed: the result's tensors take their place."""
    device = _state(lengths, tables, shares, block_size)
    requests, width = tables.shape
    blocks = shares.numel()
    out_tables, out_shares, free = tables.new_empty((requests, width)), shares.new_empty(blocks), shares.new_empty(blocks)
    ring, moves, work = lengths.new_empty(4, dtype=torch.int64), lengths.new_empty((2, blocks // 2)), shares.new_empty(blocks)
    _ebx.check(_ebx.load().ebx_kv_compact(
        lengths.data_ptr(), tables.data_ptr(), width, block_size, shares.data_ptr(), blocks, requests, out_tables.data_ptr(),
        out_shares.data_ptr(), free.data_ptr(), ring.data_ptr(), moves[0].data_ptr(), moves[1].data_ptr(), work.data_ptr(),
        4 * blocks, device, _stream(device)))
    return KVCompact(out_tables, out_shares, free, ring, KVMoves(moves[0], moves[1], ring[3:]))


def copy(pools: Sequence[KVPool], moves: KVMoves) -> None:
    """Blocks ``moves.sources`` to ``moves.targets``, codes and scales, in every pool (layers of equal sizes), in place.
    Pairs with a number that is no block are skipped; no target is another pair's source or target."""
    if not pools:
        return
    device = pools[0].device
    sources, targets, count = moves
    _refuse_ints(device, sources=(sources, torch.int32), targets=(targets, torch.int32), count=(count, torch.int64))
    if sources.numel() != targets.numel() or (count is not None and count.numel() < 1):
        raise ValueError("sources and targets must be as many, and count one number")
    array = (_ebx.KVPool * len(pools))(*(p._c for p in pools))
    _ebx.check(_ebx.load().ebx_kv_copy(array, len(pools), sources.data_ptr(), targets.data_ptr(),
                                       None if count is None else count.data_ptr(), sources.numel(), _stream(device)))


__all__ = ["KVCompact", "KVFork", "KVMoves", "compact", "copy", "fork"]
