"""Serving over a paged key-value cache held in 8 bits (no reference file: vLLM's
block manager and attention play this part there).

A layer's cache is a pool of blocks of 16, 32, 64 or 128 positions: e4m3 codes, each
block and KV head with a power of two as scale (``PagedCache``). A sequence owns the
blocks that its row of ``tables`` (int32 [batch, width], below 0 where it has none)
names in order of position; a block serves one sequence, and the same block of every
layer. ``free`` (int32) is a stack of the blocks that nobody owns: its first
``free_count[0]`` entries. In the order of a step:

    plan = plan_step(lengths, counts, tables, free, free_count, rows, block_size)  # once
    write_blocks(k, v, cache, plan.slots)                                    # a layer
    o = paged_attention(q, cache, tables, plan.starts, plan.lengths)         # a layer
    lengths = plan.lengths                    # where it is not -1
    release_blocks(tables, keep, free, free_count, block_size)   # finished, rolled back

The rows of a step are packed: ``counts[b]`` new tokens of sequence b (a decode's one,
a prompt's chunk, or none) from row ``starts[b]`` on. Everything that differs between
sequences is read on the device, so that a captured step serves every length and mix
of up to ``rows`` tokens. ``lengths[b] < 0`` marks an empty slot of the batch.

There is no backward pass: inputs that autograd follows are refused.
"""

from __future__ import annotations

import math
from operator import index
from typing import NamedTuple, Optional

import torch

from polarengine_vllm import _lib
from polarengine_vllm.kernels._calls import call, inputs, int64, written

# None in a torch that is too old for them: importing the package does not need them
F8, E8 = (getattr(torch, name, None) for name in ("float8_e4m3fn", "float8_e8m0fnu"))
BLOCK_SIZES = (16, 32, 64, 128)


class PagedCache(NamedTuple):
    """One layer's cache. Blocks may be strided (a slice of a larger pool); what
    belongs to a block is contiguous."""

    k: torch.Tensor        # float8_e4m3fn [blocks, kv_heads, block_size, head_dim]
    v: torch.Tensor        # float8_e4m3fn [blocks, kv_heads, head_dim, block_size]
    k_scale: torch.Tensor  # float8_e8m0fnu [blocks, kv_heads]
    v_scale: torch.Tensor


class StepPlan(NamedTuple):
    """What the layers of one step share, int64."""

    starts: torch.Tensor     # [batch + 1]: first row of each sequence, at most `rows`
    positions: torch.Tensor  # [rows]: position of each row in its sequence, or -1
    slots: torch.Tensor      # [rows]: block * block_size + place in the block, or -1
    lengths: torch.Tensor    # [batch]: positions after the step; -1: empty or no room


def new_cache(blocks: int, kv_heads: int, block_size: int, head_dim: int, device) -> PagedCache:
    """A layer's cache for ``blocks`` blocks."""
    if F8 is None or E8 is None:
        raise RuntimeError("the paged cache needs a torch with float8_e4m3fn and float8_e8m0fnu")
    _block_size(block_size)
    if blocks < 1 or kv_heads < 1 or head_dim not in (64, 128, 256):
        raise ValueError(f"a cache has at least one block and KV head of 64, 128 or 256 dimensions, "
                         f"got {blocks}, {kv_heads} and {head_dim}")
    return PagedCache(
        torch.zeros(blocks, kv_heads, block_size, head_dim, dtype=torch.uint8, device=device).view(F8),
        torch.zeros(blocks, kv_heads, head_dim, block_size, dtype=torch.uint8, device=device).view(F8),
        *(torch.full((blocks, kv_heads), 127, dtype=torch.uint8, device=device).view(E8)
          for _ in range(2)))


class PagedPool:
    """The caches of a model's layers, which share one set of blocks: tables, the stack
    of free blocks and the sequences' lengths, for up to ``batch`` sequences of
    ``max_len`` positions (rounded down to whole blocks) at a time."""

    def __init__(self, layers: int, blocks: int, kv_heads: int, head_dim: int, batch: int,
                 max_len: int, device, block_size: int = 64) -> None:
        _block_size(block_size)
        if batch < 1 or max_len < block_size:
            raise ValueError(f"a pool has room for at least one sequence of a block, got {batch} of "
                             f"{max_len}")
        self.block_size = block_size
        self.caches = [new_cache(blocks, kv_heads, block_size, head_dim, device) for _ in range(layers)]
        self.tables = torch.full((batch, max_len // block_size), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), blocks, dtype=torch.int64, device=device)
        self.lengths = torch.full((batch,), -1, dtype=torch.int64, device=device)  # -1: empty slot

    def plan(self, counts: torch.Tensor, rows: int) -> StepPlan:
        """``plan_step`` for ``counts[b]`` new tokens of each sequence; lengths follow
        where there was room."""
        plan = plan_step(self.lengths, counts, self.tables, self.free, self.free_count, rows,
                         self.block_size)
        torch.where(plan.lengths >= 0, plan.lengths, self.lengths, out=self.lengths)
        return plan

    def keep(self, lengths: torch.Tensor) -> None:
        """Each sequence's first ``lengths[b]`` positions stay (int64 [batch]), as many as
        it has, and its other blocks are free again: 0 begins a new sequence, below 0
        leaves an empty slot. An empty slot stays one unless it is given 0."""
        release_blocks(self.tables, lengths.clamp(min=0), self.free, self.free_count, self.block_size)
        # of an empty slot, -1, the smaller of both but for a 0
        self.lengths.copy_(torch.minimum(lengths, self.lengths).masked_fill_(lengths == 0, 0))


def _block_size(t: int) -> None:
    if t not in BLOCK_SIZES:
        raise ValueError(f"blocks hold {BLOCK_SIZES} positions, got {t}")


def _cache(cache: PagedCache):
    """(the library's arguments of a cache up to its sizes, shape of the keys)."""
    k, v, ks, vs = cache
    shape, pair = k.shape, ks.shape
    if len(shape) != 4 or v.shape != (shape[0], shape[1], shape[3], shape[2]):
        raise ValueError(f"codes must be [blocks, kv_heads, block_size, head_dim] and [.., head_dim, "
                         f"block_size], got {list(shape)} and {list(v.shape)}")
    blocks, heads, t, d = shape
    if pair != (blocks, heads) or vs.shape != pair:
        raise ValueError(f"scales must be {list(shape[:2])}, got {list(pair)} and {list(vs.shape)}")
    if not (k.dtype is v.dtype is F8 and ks.dtype is vs.dtype is E8):
        raise TypeError(f"codes must be {F8} and scales {E8}, got {k.dtype}, {v.dtype}, {ks.dtype} "
                        f"and {vs.dtype}")
    _block_size(t)
    if not blocks or not heads:
        raise ValueError(f"a cache has at least one block and KV head, got {list(shape)}")
    sk, sv, ss, head = k.stride(), v.stride(), ks.stride(), t * d
    if (sk[1:] != (head, d, 1) or sv[1:] != (head, t, 1) or ss[1] != 1 or ss != vs.stride()
            or sk[0] < heads * head or sv[0] < heads * head or ss[0] < heads):
        # a stride along one element says nothing
        sk, sv, ss = _block_stride(k), _block_stride(v), _block_stride(ks)
        if ss != _block_stride(vs):
            raise ValueError("both scales of a cache have one stride of blocks")
    return (k.data_ptr(), sk[0], v.data_ptr(), sv[0], ks.data_ptr(), vs.data_ptr(), ss[0], blocks,
            heads, t, d), shape


def _block_stride(x: torch.Tensor):
    """(stride of blocks,) of a part of a cache that has blocks of contiguous memory."""
    part = x[0].numel()
    stride = x.stride(0) if x.shape[0] > 1 else part
    if not x[0].is_contiguous() or stride < part:
        raise ValueError(f"what belongs to a block must be contiguous, and blocks may not overlap: got "
                         f"strides {x.stride()} for {list(x.shape)}")
    return (stride,)


def _tables(tables: torch.Tensor, batch: int, change: bool) -> torch.Tensor:
    if tables.dtype is not torch.int32:
        raise TypeError(f"tables must be int32, got {tables.dtype}")
    if tables.dim() != 2 or tables.shape[0] != batch or not tables.shape[1]:
        raise ValueError(f"tables must be [{batch}, width], got {list(tables.shape)}")
    width = tables.shape[1]
    if (width > 1 and tables.stride(1) != 1) or (batch > 1 and tables.stride(0) < width):
        if change:
            raise ValueError(f"tables must have contiguous rows that do not overlap, got strides "
                             f"{tables.stride()}")
        tables = tables.contiguous()
    return tables


def _row_stride(tables: torch.Tensor) -> int:
    return tables.stride(0) if tables.shape[0] > 1 else tables.shape[1]


def _pool(tables, free, free_count, batch, block_size):
    _block_size(block_size)
    _tables(tables, batch, True)
    if free.dtype is not torch.int32 or free_count.dtype is not torch.int64:
        raise TypeError(f"free must be int32 and free_count int64, got {free.dtype} and "
                        f"{free_count.dtype}")
    if free.dim() != 1 or not free.is_contiguous() or not free.numel() or free_count.numel() != 1:
        raise ValueError(f"free must be a contiguous stack of blocks and free_count one number, got "
                         f"{list(free.shape)} and {list(free_count.shape)}")
    return (_row_stride(tables), batch, tables.shape[1])


def plan_step(lengths: torch.Tensor, counts: torch.Tensor, tables: torch.Tensor,
              free: torch.Tensor, free_count: torch.Tensor, rows: int,
              block_size: int) -> StepPlan:
    """Room for ``counts[b]`` more positions of each sequence of ``lengths[b]`` (int64
    [batch]), and where the step's rows belong.

    Blocks that a sequence lacks for its new positions come off the stack's end, in
    order of sequence and position; ``tables`` and ``free_count`` change in place. A
    sequence gets all that it asks for or nothing: nothing where its rows pass
    ``rows`` (what the step's tensors hold), its positions its table, or the blocks
    asked for up to and with it the stack. At most 4096 sequences, 2^24 rows."""
    dev = inputs(lengths, counts, tables, free, free_count)
    if lengths.dim() != 1:
        raise ValueError(f"lengths must be [batch], got {list(lengths.shape)}")
    batch = lengths.shape[0]
    pool = _pool(tables, free, free_count, batch, block_size)
    if rows < 0:
        raise ValueError(f"rows must be at least 0, got {rows}")
    lengths, counts = int64(lengths, (batch,), "lengths"), int64(counts, (batch,), "counts")
    out = torch.empty(2 * batch + 1 + 2 * rows, dtype=torch.int64, device=dev)
    positions, slots, starts, after = out.split_with_sizes((rows, rows, batch + 1, batch))
    if not batch:
        positions.fill_(-1), slots.fill_(-1), starts.zero_()
        return StepPlan(starts, positions, slots, after)
    call("pe_plan_step", dev, lengths.data_ptr(), counts.data_ptr(), tables.data_ptr(), *pool,
         free.data_ptr(), free.numel(), free_count.data_ptr(), rows, block_size, starts.data_ptr(),
         positions.data_ptr(), slots.data_ptr(), after.data_ptr())
    written(tables, free_count)
    return StepPlan(starts, positions, slots, after)


def release_blocks(tables: torch.Tensor, keep: torch.Tensor, free: torch.Tensor,
                   free_count: torch.Tensor, block_size: int) -> None:
    """The blocks of each sequence behind its first ``keep[b]`` positions (int64
    [batch]; 0: all, below 0: none), up to its first entry below 0, back to the stack;
    -1 takes their place in ``tables``. What a plan took goes back as it was."""
    dev = inputs(tables, keep, free, free_count)
    if keep.dim() != 1:
        raise ValueError(f"keep must be [batch], got {list(keep.shape)}")
    batch = keep.shape[0]
    pool = _pool(tables, free, free_count, batch, block_size)
    keep = int64(keep, (batch,), "keep")
    if not batch:
        return
    call("pe_release_blocks", dev, tables.data_ptr(), *pool, keep.data_ptr(), free.data_ptr(),
         free.numel(), free_count.data_ptr(), block_size)
    written(tables, free, free_count)


def check_sight(window: Optional[int], sinks: int) -> None:
    """Refuses what ``paged_attention`` takes for no window and first positions."""
    if window is not None and index(window) < 1:
        raise ValueError(f"a window holds at least one position, got {window}")
    if index(sinks) < 0:
        raise ValueError(f"sinks must be at least 0, got {sinks}")


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """Rows of heads that the kernels read 16 bytes at a time."""
    st = x.stride()
    if st[2] != 1 or (st[0] | st[1]) % 8 or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format)
    return x


def write_blocks(k: torch.Tensor, v: torch.Tensor, cache: PagedCache, slots: torch.Tensor) -> None:
    """Keys and values [rows, kv_heads, head_dim] (fp16 or bf16) to ``slots`` (int64
    [rows]; outside the cache: left out).

    A run, neighbouring rows whose slots rise by one within a block, gives the block
    (per head, keys and values apart) the smallest scale 2^e, e >= -100, that holds its
    largest finite value as at most 448 2^e, and never a smaller one than the block
    has, unless the run begins at the block's first slot. Codes that the block holds
    already are rounded to a grown scale. Values are rounded once, to nearest even;
    infinite ones and NaN become NaN. Only one run of a call may go to a block."""
    dev = inputs(k, v, slots, *cache)
    code = _lib.act_dtype(k)
    args, shape = _cache(cache)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (shape[1], shape[3]) or v.dtype is not k.dtype:
        raise ValueError(f"keys and values must be [rows, {shape[1]}, {shape[3]}] of one type, got "
                         f"{list(k.shape)} {k.dtype} and {list(v.shape)} {v.dtype}")
    if cache.k.data_ptr() == cache.v.data_ptr() or cache.k_scale.data_ptr() == cache.v_scale.data_ptr():
        raise ValueError("keys and values of the cache are the same memory")
    rows = k.shape[0]
    slots = int64(slots, (rows,), "slots")
    if not rows:
        return
    k, v = _rows16(k), _rows16(v)
    call("pe_write_blocks", dev, k.data_ptr(), v.data_ptr(), code, rows, *k.stride()[:2],
         *v.stride()[:2], slots.data_ptr(), *args)
    written(*cache)


def paged_attention(q: torch.Tensor, cache: PagedCache, tables: torch.Tensor, starts: torch.Tensor,
                    lengths: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                    scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q K^T) V of packed rows q [rows, heads, head_dim] (fp16 or bf16)
    over the cache: the rows of sequence b begin at ``starts[b]`` (int64 [batch + 1]),
    its last one is at position ``lengths[b] - 1`` (int64 [batch]). A row sees the
    positions up to its own; with a ``window`` the last ``window`` of them and the
    first ``sinks`` of the sequence. scale: at least 0, 1 / sqrt(head_dim) if not given.

    Zeros for rows outside all sequences, of a sequence with ``lengths[b] < 0`` and
    where nothing is in sight; positions whose block is none of the cache's are not
    seen. Scores, softmax statistics and sums in fp32; a probability times its value's
    scale is rounded to fp16 once, relative to the row's largest such product: 2^-20 of
    that keeps all of its bits, what is below 2^-31 of it may be dropped."""
    dev = inputs(q, tables, starts, lengths, *cache)
    code = _lib.act_dtype(q)
    args, shape = _cache(cache)
    if q.dim() != 3 or q.shape[2] != shape[3] or not q.shape[1] or q.shape[1] % shape[1]:
        raise ValueError(f"q must be [rows, heads, {shape[3]}] with a multiple of {shape[1]} heads, got "
                         f"{list(q.shape)}")
    if lengths.dim() != 1:
        raise ValueError(f"lengths must be [batch], got {list(lengths.shape)}")
    check_sight(window, sinks)
    (rows, heads, dim), batch = q.shape, lengths.shape[0]
    tables = _tables(tables, batch, False)
    starts, lengths = int64(starts, (batch + 1,), "starts"), int64(lengths, (batch,), "lengths")
    if not rows or not batch:
        return torch.zeros(rows, heads, dim, dtype=q.dtype, device=dev)
    if q.stride(1) != dim or q.stride(2) != 1 or q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = q.new_empty((rows, heads, dim))
    width = tables.shape[1]
    size = _lib.workspace_size("pe_paged_attention_workspace_size", rows, batch, heads, shape[1], dim,
                               width * shape[2])
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    call("pe_paged_attention", dev, q.data_ptr(), code, q.stride(0), rows, heads, *args,
         tables.data_ptr(), _row_stride(tables), batch, width, starts.data_ptr(), lengths.data_ptr(),
         min(window or 0, 1 << 40), min(sinks, 1 << 40), 1.0 / math.sqrt(dim) if scale is None else scale, out.data_ptr(),
         _lib.ptr(ws), size)
    return out
