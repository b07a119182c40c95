"""An 8-bit paged key/value cache for the decoders that ElasticBit compresses.

The weights of a compressed model are read as integer codes; at serving lengths the keys and
values are the larger part of what a step reads, so they are kept as codes too: a block of 16 to
128 tokens of one head is int8 under one fp32 scale (value = code * scale), half the bytes of a
16-bit cache.  Blocks belong to requests through a block table, so that ragged requests share one
pool.  Four operators (``libebx``, include/ebx.h ``ebx_kv_*``), all stream-ordered, none of which
copies anything to the host:

* ``plan``         blocks and slots of a step's new tokens, from the requests' lengths on the GPU;
* ``append``       quantises the new keys and values into their slots;
* ``attention``    new queries over the cache: decode steps, prompts, chunks, sliding windows;
* ``materialize``  keys and values back in 16 or 32 bits.

``KVCache`` holds a model's pools and tables and runs them together.  Inference only, as the rest
of the native route: no autograd.  The reference has no counterpart (its caches,
mlbricks/cache.py, are whole 16-bit tensors).
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple

import torch

from . import _ebx

BLOCK_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128)
_ROW_DTYPES = {torch.float16: 1, torch.bfloat16: 2}
_DTYPES = {torch.float32: 0, **_ROW_DTYPES}


class KVPlan(NamedTuple):
    """A step: what ``plan`` wrote (all on the GPU)."""

    lengths: torch.Tensor    # int32 [requests], tokens held once the step's are appended
    starts: torch.Tensor     # int32 [requests + 1], first token of each request in the step
    slots: torch.Tensor      # int64 [tokens], where each token goes; -1: nowhere
    positions: torch.Tensor  # int32 [tokens], its place in its request
    ring: torch.Tensor       # int64 [4]: front, back, blocks that were missing, tokens


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


# These calls are made every step and every layer, so what can be wrong is looked for in one
# expression, and told apart only when something is.
def _int_ok(t: torch.Tensor, dtype: torch.dtype, device: int) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.is_contiguous()


def _refuse_ints(device: int, **tensors) -> None:
    for name, (t, dtype) in tensors.items():
        if t is not None and not _int_ok(t, dtype, device):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor on cuda:{device}")


class KVPool:
    """One layer's cache: int8 codes [blocks, kv_heads, block_size, head_dim] and fp32 scales
    [blocks, kv_heads], of keys and of values.  Holds the tensors; copies nothing.  Scales are >= 0, or
    NaN for a block that holds a value that is not finite, as ``append`` writes them."""

    __slots__ = ("k_codes", "k_scales", "v_codes", "v_scales", "device", "_c", "_ref")

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                 v_scales: torch.Tensor) -> None:
        shape, device = k_codes.shape, k_codes.get_device()
        scales = shape[:2]
        if not (len(shape) == 4 and device >= 0 and v_codes.shape == shape and k_scales.shape == scales
                and v_scales.shape == scales and _int_ok(k_codes, torch.int8, device)
                and _int_ok(v_codes, torch.int8, device) and _int_ok(k_scales, torch.float32, device)
                and _int_ok(v_scales, torch.float32, device)):
            self._refuse(k_codes, k_scales, v_codes, v_scales)
        blocks, kv_heads, block_size, head_dim = shape
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if not 0 < blocks * kv_heads * block_size < 2**31:
            raise ValueError("need 0 < blocks * kv_heads * block_size < 2^31")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.device = device
        self._c = _ebx.KVPool(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                              blocks, kv_heads, block_size, head_dim, device, 0)
        self._ref = ctypes.byref(self._c)

    @staticmethod
    def _refuse(k_codes, k_scales, v_codes, v_scales) -> None:
        shape, device = k_codes.shape, k_codes.get_device()
        if len(shape) != 4 or device < 0:
            raise ValueError("codes must be CUDA tensors [blocks, kv_heads, block_size, head_dim]")
        for name, t, dtype, want in (("k_codes", k_codes, torch.int8, shape), ("v_codes", v_codes, torch.int8, shape),
                                     ("k_scales", k_scales, torch.float32, shape[:2]),
                                     ("v_scales", v_scales, torch.float32, shape[:2])):
            if t.shape != want or not _int_ok(t, dtype, device):
                raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(want)} on cuda:{device}")

    @classmethod
    def empty(cls, blocks: int, kv_heads: int, block_size: int, head_dim: int, device="cuda") -> "KVPool":
        """A pool whose blocks hold nothing yet."""
        shape = (blocks, kv_heads, block_size, head_dim)
        return cls(*(t for _ in "kv" for t in (torch.zeros(shape, dtype=torch.int8, device=device),
                                               torch.zeros(shape[:2], dtype=torch.float32, device=device))))

    blocks = property(lambda self: self._c.blocks)
    kv_heads = property(lambda self: self._c.kv_heads)
    block_size = property(lambda self: self._c.block_size)
    head_dim = property(lambda self: self._c.head_dim)

    def _rows(self, x: torch.Tensor, heads: int | None, name: str) -> torch.Tensor:
        """x [tokens, heads, head_dim] as the kernels read it: 16-byte aligned rows."""
        if x.dtype not in _ROW_DTYPES or x.get_device() != self.device:
            raise ValueError(f"{name} must be float16 or bfloat16 on cuda:{self.device}")
        if x.dim() != 3 or x.shape[2] != self._c.head_dim or (heads is not None and x.shape[1] != heads):
            raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, "
                             f"{self._c.head_dim}], got {tuple(x.shape)}")
        s0, s1, s2 = x.stride()
        if s2 != 1 or s0 % 8 or s1 % 8 or x.data_ptr() % 16:
            return x.clone(memory_format=torch.contiguous_format)
        return x


def _stream(device: int) -> int:
    return _RAW_STREAM(device) if _RAW_STREAM is not None else _ebx.stream_ptr(device=device)


_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device: int, kv_heads: int, head_dim: int, heads: int, tokens: int, max_new: int,
                     max_length: int) -> int:
    pool = _ebx.KVPool(16, 16, 16, 16, 1, kv_heads, BLOCK_SIZES[0], head_dim, device, 0)  # only its sizes count
    return int(_ebx.load().ebx_kv_attention_workspace_bytes(ctypes.byref(pool), heads, tokens, max_new, max_length))


def plan(past: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, ring: torch.Tensor, *,
         block_size: int, tokens: int) -> KVPlan:
    """Blocks and slots of one step, on the GPU.

    Request i holds ``past[i]`` tokens and brings ``new[i]``; ``new[i] < 0`` releases it.  Free
    blocks wait in the ring ``free`` (int32, room for every block) from ``ring[0]`` up to
    ``ring[1]``, modulo its size.  In order, each request takes the blocks that it lacks into its
    row of ``tables`` (written in place) -- or nothing, if they are not all there, the row is too
    short, or its tokens do not fit ``tokens``: they then get slot -1, its length stays, and ``ring[2]``
    of the result counts the blocks that it needed.  Nobody overtakes: behind the first request that
    finds too few blocks, no other gets one in this step; those that need none go on.  Refused tokens
    keep their rows (``starts``), so what ``attention`` returns there means nothing: leave out rows with
    slot -1.  Released blocks join the ring's back.  ``tokens`` is the
    room for slots and positions: the sum of the new tokens, or more (the rest is slot -1, position 0);
    ``ring[3]`` of the result is that sum, so ``ring[3] > tokens`` says that requests were refused for
    want of room.

    The inputs ``past`` and ``ring`` are not changed; the next step takes the result's ``lengths``
    and ``ring`` in their place."""
    device = past.get_device()
    if device < 0:
        raise ValueError("plan needs CUDA tensors")
    int32, requests = torch.int32, past.numel()
    if not (_int_ok(past, int32, device) and _int_ok(new, int32, device) and _int_ok(tables, int32, device)
            and _int_ok(free, int32, device) and _int_ok(ring, torch.int64, device)):
        _refuse_ints(device, past=(past, int32), new=(new, int32), tables=(tables, int32), free=(free, int32),
                     ring=(ring, torch.int64))
    if new.numel() != requests or tables.dim() != 2 or tables.shape[0] != requests:
        raise ValueError("past, new and the rows of tables must be as many")
    if ring.numel() < 2 or tokens < 0:
        raise ValueError("ring holds at least its front and back, and tokens >= 0")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    # new_empty: the cheapest way to a tensor, and this call is made every step
    lengths, starts, positions = past.new_empty(requests), past.new_empty(requests + 1), past.new_empty(tokens)
    slots, out = ring.new_empty(tokens), ring.new_empty(4)
    st = _ebx.load().ebx_kv_plan(
        past.data_ptr(), new.data_ptr(), requests, tables.data_ptr(), tables.shape[1], block_size,
        free.data_ptr(), free.numel(), ring.data_ptr(), out.data_ptr(), lengths.data_ptr(), starts.data_ptr(),
        slots.data_ptr(), positions.data_ptr(), tokens, device, _stream(device))
    if st:
        _ebx.check(st)
    return KVPlan(lengths, starts, slots, positions, out)


def append(k: torch.Tensor, v: torch.Tensor, pool: KVPool, slots: torch.Tensor) -> None:
    """Quantise new keys and values [tokens, kv_heads, head_dim] (fp16 or bf16, any strides) into
    their slots, in place.  For each block and head the scale is max(old, max |x| / 127) and a code
    rint(x / scale); tokens that the block held before move to a larger scale.  Tokens with slot -1
    are skipped; a value that is not finite makes the scale of its block NaN.  The tokens of one
    block are consecutive, behind all that the block holds (as ``plan`` lays them)."""
    heads = pool._c.kv_heads
    k, v = pool._rows(k, heads, "k"), pool._rows(v, heads, "v")
    tokens = k.shape[0]
    if v.shape[0] != tokens or v.dtype is not k.dtype:
        raise ValueError("k and v must have the same tokens and dtype")
    if not _int_ok(slots, torch.int64, pool.device):
        _refuse_ints(pool.device, slots=(slots, torch.int64))
    if slots.numel() != tokens:
        raise ValueError("slots must have one entry for each token")
    if tokens == 0:
        return
    st = _ebx.load().ebx_kv_append(
        pool._ref, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
        slots.data_ptr(), tokens, _ROW_DTYPES[k.dtype], _stream(pool.device))
    if st:
        _ebx.check(st)


def materialize(pool: KVPool, tables: torch.Tensor, starts: torch.Tensor, *, first: torch.Tensor | None = None,
                tokens: int, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [tokens, kv_heads, head_dim] as code * scale, rounded once to ``dtype``:
    rows starts[i] .. starts[i + 1] - 1 are the places first[i] (default 0) on of request i.  The caller
    keeps them within what the request holds: behind that the table may name other requests' blocks."""
    if dtype not in _DTYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    requests = starts.numel() - 1
    int32, device = torch.int32, pool.device
    if not (_int_ok(starts, int32, device) and _int_ok(tables, int32, device)
            and (first is None or _int_ok(first, int32, device))):
        _refuse_ints(device, starts=(starts, int32), tables=(tables, int32), first=(first, int32))
    if requests < 0 or tables.dim() != 2 or tables.shape[0] != requests or tokens < 0:
        raise ValueError("tables must have a row, and starts an entry, for each request (and one more); tokens >= 0")
    if first is not None and first.numel() != requests:
        raise ValueError("first must have one entry for each request")
    shape = (tokens, pool._c.kv_heads, pool._c.head_dim)
    k, v = starts.new_empty(shape, dtype=dtype), starts.new_empty(shape, dtype=dtype)
    st = _ebx.load().ebx_kv_materialize(
        pool._ref, tables.data_ptr(), tables.shape[1], starts.data_ptr(), None if first is None else first.data_ptr(),
        requests, tokens, _DTYPES[dtype], k.data_ptr(), v.data_ptr(), _stream(device))
    if st:
        _ebx.check(st)
    return k, v


def attention(q: torch.Tensor, pool: KVPool, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, *,
              scale: float | None = None, causal: bool = True, window: int = 0, first: torch.Tensor | None = None,
              max_new: int = 0, max_length: int = 0, out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of new queries [tokens, heads, head_dim] (fp16 or bf16, any strides) over the cache.

    Request i's queries are rows starts[i] .. starts[i + 1] - 1, at the last positions of its
    lengths[i] tokens; heads / kv_heads query heads share a key/value head.  A query at position p
    sees the keys j < lengths[i] with j >= first[i] (if given), j <= p (``causal``) and
    j > p - window (``window`` > 0).  A query that sees nothing gets 0 (log-sum-exp -infinity); rows
    of no request are left as they are, and ``out``, if given, is not q's memory.  ``scale`` defaults to
    1 / sqrt(head_dim).  ``max_new`` and
    ``max_length``, where the caller knows the largest number of new tokens and the largest length,
    choose the kernel: they change the order of sums, not the formula.  Without ``max_new`` a batch of
    49 rows (tokens * heads / kv_heads) and more is taken for a prompt, which costs single tokens about three
    times their time.  Returns out, or (out, lse [tokens, heads] fp32)."""
    q = pool._rows(q, None, "q")
    device = pool.device
    tokens, heads, dim = q.shape
    requests = lengths.numel()
    int32 = torch.int32
    if not (_int_ok(tables, int32, device) and _int_ok(lengths, int32, device) and _int_ok(starts, int32, device)
            and (first is None or _int_ok(first, int32, device))):
        _refuse_ints(device, tables=(tables, int32), lengths=(lengths, int32), starts=(starts, int32), first=(first, int32))
    if heads == 0 or heads % pool._c.kv_heads:
        raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({pool._c.kv_heads})")
    if starts.numel() != requests + 1 or tables.dim() != 2 or tables.shape[0] != requests:
        raise ValueError("lengths and the rows of tables must be as many, and starts one more")
    if first is not None and first.numel() != requests:
        raise ValueError("first must have one entry for each request")
    if out is None:
        out = q.new_empty((tokens, heads, dim))
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != device or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape and dtype")
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    if tokens and requests:
        lib = _ebx.load()
        nbytes = _workspace_bytes(device, pool._c.kv_heads, dim, heads, tokens, max_new, max_length)
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        st = lib.ebx_kv_attention(
            pool._ref, q.data_ptr(), q.stride(0), q.stride(1), heads, _ROW_DTYPES[q.dtype], tables.data_ptr(),
            tables.shape[1], lengths.data_ptr(), starts.data_ptr(), None if first is None else first.data_ptr(),
            requests, tokens, causal, window, 1.0 / math.sqrt(dim) if scale is None else scale, max_new, max_length,
            out.data_ptr(), None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
            _stream(device))
        if st:
            _ebx.check(st)
    return out if lse is None else (out, lse)


class KVCache:
    """Pools, block table and free ring of a model with ``layers`` layers, for up to ``requests``
    requests of up to ``max_length`` tokens at a time.

    A step is ``plan(new)`` and then, layer by layer, ``append`` and ``attention``; ``new[i]`` is the
    number of tokens that request i brings (0: it rests, -1: it is done and gives its blocks back).
    The state stays in the same tensors, so a step with fixed sizes can be captured in a CUDA graph
    and replayed.  One stream at a time; more than one needs the caller's events."""

    def __init__(self, layers: int, blocks: int, kv_heads: int, head_dim: int, *, requests: int, max_length: int,
                 block_size: int = 64, device="cuda") -> None:
        _check(layers > 0 and requests > 0 and max_length > 0, "layers, requests and max_length must be positive")
        self.pools = [KVPool.empty(blocks, kv_heads, block_size, head_dim, device) for _ in range(layers)]
        self.block_size, self.max_length = block_size, max_length
        where = self.pools[0].k_codes.device
        self.tables = torch.full((requests, -(-max_length // block_size)), -1, dtype=torch.int32, device=where)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=where)
        self.free = torch.arange(blocks, dtype=torch.int32, device=where)
        self.ring = torch.tensor([0, blocks, 0, 0], dtype=torch.int64, device=where)
        self.step: KVPlan | None = None
        self._max_new = 0

    def plan(self, new, tokens: int | None = None, max_new: int | None = None) -> KVPlan:
        """Blocks and slots for a step.  ``new``: a list, or an int32 tensor on the GPU with
        ``tokens`` (room for all its tokens; requests that end past it are refused) and ``max_new``, without which ``attention`` takes a batch
        of single tokens for a prompt.  ``ring[2]`` of the result is the number of blocks that refused requests
        needed: they keep their length, their tokens have slot -1, and their rows of ``attention`` mean nothing."""
        if not isinstance(new, torch.Tensor):
            counts = [max(int(n), 0) for n in new]
            tokens, max_new = sum(counts), max(counts, default=0)
            new = torch.tensor([int(n) for n in new], dtype=torch.int32).to(self.lengths.device, non_blocking=True)
        _check(tokens is not None, "a tensor of new tokens needs `tokens`")
        self.step = plan(self.lengths, new, self.tables, self.free, self.ring, block_size=self.block_size, tokens=tokens)
        self.lengths.copy_(self.step.lengths)
        self.ring.copy_(self.step.ring)
        self._max_new = max_new or 0
        return self.step

    def _planned(self) -> KVPlan:
        if self.step is None:
            raise RuntimeError("KVCache: plan a step first")
        return self.step

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's keys and values [tokens, kv_heads, head_dim] into the layer's pool."""
        append(k, v, self.pools[layer], self._planned().slots)

    def attention(self, layer: int, q: torch.Tensor, **options):
        """The step's queries [tokens, heads, head_dim] over the layer's cache (``attention``'s options)."""
        step = self._planned()
        return attention(q, self.pools[layer], self.tables, step.lengths, step.starts, max_new=self._max_new,
                         max_length=self.max_length, **options)

    def materialize(self, layer: int, starts: torch.Tensor, *, tokens: int, first: torch.Tensor | None = None,
                    dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values that the layer holds (``materialize``'s arguments)."""
        return materialize(self.pools[layer], self.tables, starts, first=first, tokens=tokens, dtype=dtype)


__all__ = ["BLOCK_SIZES", "HEAD_DIMS", "KVCache", "KVPlan", "KVPool", "append", "attention", "materialize", "plan"]
