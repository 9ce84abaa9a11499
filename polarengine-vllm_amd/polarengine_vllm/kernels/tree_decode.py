"""A decode step with several drafted tokens per sequence (speculative decoding;
no reference file: vLLM's model runner plays this part there).

A sequence's step has n nodes, 1 <= n <= 64: node 0 is its last token, node i > 0
a drafted token that follows node ``parents[i]`` < i; a chain has ``parents[i] =
i - 1``. Node i's key and value go to cache slot ``lengths[b] + i``; the slots
below ``lengths[b]`` hold the sequence so far. In the order of a step:

    plan = tree_plan(parents, lengths)                      # once
    q = qk_norm_rope_write(qkv, ..., plan.positions, k_cache, v_cache, lengths)  # a layer
    o = tree_attention(q, k_cache, v_cache, lengths, plan.masks)                 # a layer
    tokens, path, count = verify_drafts(logits, drafts, uniforms, parents=parents)
    keep_accepted(k_caches, v_caches, lengths, path, count)  # all layers
    lengths += count

Everything that differs between sequences is read on the device, so a captured
step serves every length, tree and outcome. ``lengths[b] < 0``, or too long for the
cache to hold n more, marks an empty slot of the batch: the attention gives it
zeros, and nothing of it is written or moved. (The queries follow the positions
alone: zeros where the table has none, as for the plan's -1.) ``verify_drafts``
knows an empty slot by its node 0's token. A node whose parent is no earlier
existing node is absent (a padded place of a smaller tree).

Caches are [batch, kv_heads, positions, head_dim] views, fp16 or bf16: values with
the dimension contiguous, keys with the dimension or the position contiguous (the
latter is ``k_cache.transpose(-1, -2)`` of a [.., head_dim, positions] tensor, as
``DecodeRunner`` holds its keys). Rows with the dimension contiguous are read 16
bytes at a time: 16-byte aligned, strides multiples of 8. Written caches may not
overlap themselves. There is no backward pass: inputs that autograd follows are
refused.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from polarengine_vllm import _lib
from polarengine_vllm.kernels._calls import (call as _call, inputs as _inputs, int64 as _int64,
                                             written as _written)

MAX_NODES = 64


class TreePlan(NamedTuple):
    """What the layers of one step share: int64 [batch, n]."""

    positions: torch.Tensor  # of each node; -1 for absent nodes and where lengths[b] < 0
    masks: torch.Tensor      # bit j of node i's word: j is i or an ancestor of i


def _per_node(t: torch.Tensor, batch: int, n: int, name: str) -> Tuple[torch.Tensor, int]:
    """An int64 [batch, n] tensor, or [n] for all sequences alike, and its row stride."""
    if t.dtype is not torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.shape == (n,):
        return t.contiguous(), 0
    if t.shape != (batch, n):
        raise ValueError(f"{name} must be [{n}] or [{batch}, {n}], got {list(t.shape)}")
    if n > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _nodes(n: int) -> None:
    if not 1 <= n <= MAX_NODES:
        raise ValueError(f"a step takes 1 to {MAX_NODES} nodes per sequence, got {n}")


def _strides(t: torch.Tensor):
    """Element strides of a cache [.., positions, head_dim]. A stride along one element
    says nothing: 0, but 1 for the one position of keys by dimension."""
    st, shape = t.stride(), t.shape
    if 1 in shape:
        st = [0 if n == 1 else s for s, n in zip(st, shape)]
        if shape[-2] == 1 and st[-1] != 1:
            st[-2] = 1
    return st


def _caches(k: torch.Tensor, v: torch.Tensor, dtype: torch.dtype):
    """Shape and element strides of a key and a value cache."""
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"caches must be [batch, kv_heads, positions, head_dim] alike, got "
                         f"{list(k.shape)} and {list(v.shape)}")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError(f"caches must be {dtype} as the queries, got {k.dtype} and {v.dtype}")
    ks, vs, shape = _strides(k), _strides(v), k.shape
    if vs[3] != 1 or (ks[3] != 1 and ks[2] != 1):
        raise ValueError("values must have the dimension contiguous, keys the dimension or the "
                         f"position; got strides {vs} and {ks}")
    return shape, ks, vs


def _writable(t: torch.Tensor, name: str) -> None:
    """Refuses views whose elements may share memory."""
    st, n = t.stride(), t.shape
    if len(n) == 4:  # rows or columns of a head, one head after the other: the usual layouts
        low, high = (2, 3) if st[2] == 1 else (3, 2)
        if (st[low] == 1 and st[high] >= n[low] and st[1] >= st[high] * n[high]
                and st[0] >= st[1] * n[1]):
            return
    span = 1
    for stride, size in sorted(zip(st, n)):
        if size > 1:
            if stride < span:
                raise ValueError(f"{name} overlaps itself (shape {list(n)}, strides {st}): it "
                                 f"cannot be written")
            span += stride * (size - 1)


def _apart(k: torch.Tensor, v: torch.Tensor) -> None:
    if k.numel() and k.data_ptr() == v.data_ptr():
        raise ValueError("k_cache and v_cache are the same memory")


def tree_plan(parents: torch.Tensor, lengths: torch.Tensor) -> TreePlan:
    """Positions and ancestor masks of a step's nodes: parents int64 [batch, n], or
    [n] for one tree for all, lengths int64 [batch]."""
    dev = _inputs(parents, lengths)
    if lengths.dim() != 1 or parents.dim() not in (1, 2):
        raise ValueError(f"parents must be [n] or [batch, n] and lengths [batch], got "
                         f"{list(parents.shape)} and {list(lengths.shape)}")
    batch, n = lengths.shape[0], parents.shape[-1]
    _nodes(n)
    parents, stride = _per_node(parents, batch, n, "parents")
    lengths = _int64(lengths, (batch,), "lengths")
    positions = torch.empty(batch, n, dtype=torch.int64, device=dev)
    masks = torch.empty(batch, n, dtype=torch.int64, device=dev)
    if not batch:
        return TreePlan(positions, masks)
    _call("pe_tree_plan", dev, parents.data_ptr(), stride, lengths.data_ptr(), batch, n,
          positions.data_ptr(), masks.data_ptr())
    return TreePlan(positions, masks)


def _rope_inputs(qkv, heads, kv_heads, rope, positions, q_weight, k_weight):
    """Checked inputs of the two norm + rotary calls: (rows, head_dim, qkv, rope,
    positions, weights)."""
    code = _lib.act_dtype(qkv)
    per = heads + 2 * kv_heads
    if qkv.dim() != 2 or heads < 1 or kv_heads < 1 or qkv.shape[1] % per:
        raise ValueError(f"qkv must be [rows, (heads + 2 kv_heads) * head_dim] for {heads} and "
                         f"{kv_heads} heads, got {list(qkv.shape)}")
    rows, cols = qkv.shape
    dim = cols // per
    ld, one = qkv.stride()
    if one != 1 or ld % 8 or ld < cols or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    if rope.dtype is not torch.float32 or rope.dim() != 2:
        raise TypeError(f"rope must be a float32 [positions, rotary dims] table, got {rope.dtype} "
                        f"of {list(rope.shape)}")
    if positions.dtype is not torch.int64:
        raise TypeError(f"positions must be int64, got {positions.dtype}")
    if positions.numel() != rows:
        raise ValueError(f"positions must name {rows} rows, got {list(positions.shape)}")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype is not qkv.dtype or w.shape != (dim,)):
            raise ValueError(f"norm weights must be {qkv.dtype} of [{dim}], got {w.dtype} of "
                             f"{list(w.shape)}")
    return (rows, dim, code, qkv, _whole(rope), positions.contiguous(),
            None if q_weight is None else _whole(q_weight),
            None if k_weight is None else _whole(k_weight))


def _whole(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, 16-byte aligned."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def qk_norm_rope(qkv: torch.Tensor, heads: int, kv_heads: int, rope: torch.Tensor,
                 positions: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries [rows, heads, head_dim] and keys [rows, kv_heads, head_dim] of qkv
    [rows, (heads + 2 kv_heads) * head_dim] (fp16 or bf16; head_dim 64, 128 or
    256), RMS-normed per head with the weights [head_dim] that are given, then
    rotated: dimensions j and j + r / 2 of the first r by the angles of row
    positions[row] of ``rope`` float32 [table rows, r], cosines then sines, r a
    multiple of 16. In 64 bits, rounded once (the products of a value and its
    weight have to lie in fp32's range); zeros where the position is outside the
    table. ``positions`` int64, one a row in any shape."""
    dev = _inputs(qkv, rope, positions, q_weight, k_weight)
    rows, dim, code, qkv, rope, positions, qw, kw = _rope_inputs(
        qkv, heads, kv_heads, rope, positions, q_weight, k_weight)
    q = torch.empty(rows, heads, dim, dtype=qkv.dtype, device=dev)
    k = torch.empty(rows, kv_heads, dim, dtype=qkv.dtype, device=dev)
    if not rows:
        return q, k
    _call("pe_qk_norm_rope", dev, qkv.data_ptr(), code, rows, qkv.stride(0), heads, kv_heads, dim,
          rope.data_ptr(), rope.shape[0], rope.shape[1], positions.data_ptr(), _lib.ptr(qw),
          _lib.ptr(kw), eps, q.data_ptr(), k.data_ptr())
    return q, k


def qk_norm_rope_write(qkv: torch.Tensor, heads: int, kv_heads: int, rope: torch.Tensor,
                       positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       lengths: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                       k_weight: Optional[torch.Tensor] = None,
                       eps: float = 1e-6) -> torch.Tensor:
    """The same for the n rows of each sequence (any n: a step's nodes, a prompt),
    keys and values written to slots ``lengths[b] + i`` of the caches; returns the
    queries. Rows whose position is outside the table, and those of a sequence whose
    cache has no room for n more, leave their slots as they were."""
    dev = _inputs(qkv, rope, positions, k_cache, v_cache, lengths, q_weight, k_weight)
    rows, dim, code, qkv, rope, positions, qw, kw = _rope_inputs(
        qkv, heads, kv_heads, rope, positions, q_weight, k_weight)
    shape, ks, vs = _caches(k_cache, v_cache, qkv.dtype)
    batch = shape[0]
    if shape[1] != kv_heads or shape[3] != dim:
        raise ValueError(f"caches of {kv_heads} heads of {dim} are needed, got {list(shape)}")
    lengths = _int64(lengths, (batch,), "lengths")
    if (rows % batch if batch else rows):
        raise ValueError(f"{rows} rows do not go into {batch} sequences")
    _writable(k_cache, "k_cache")
    _writable(v_cache, "v_cache")
    if rows:
        _apart(k_cache, v_cache)
    q = torch.empty(rows, heads, dim, dtype=qkv.dtype, device=dev)
    if rows:
        _call("pe_qk_norm_rope_write", dev, qkv.data_ptr(), code, batch, rows // batch,
              qkv.stride(0), heads, kv_heads, dim, rope.data_ptr(), rope.shape[0], rope.shape[1],
              positions.data_ptr(), _lib.ptr(qw), _lib.ptr(kw), eps, q.data_ptr(),
              k_cache.data_ptr(), *ks, v_cache.data_ptr(), *vs[:3], lengths.data_ptr(), shape[2])
        _written(k_cache, v_cache)
    return q


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   lengths: torch.Tensor, masks: torch.Tensor,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the nodes' queries q [batch, n, heads, head_dim] (heads a
    multiple of the cache's; head_dim 64, 128 or 256): node i sees the positions
    below ``lengths[b]`` and the slots ``lengths[b] + j`` of the bits j < n of its
    mask (int64 [batch, n], or [n] for all). Scores, softmax statistics and sums in
    fp32; the probabilities are rounded to the queries' type for the product with the
    values, where fp16 loses bits of those below 2^-21 of a row's largest and all of
    those below 2^-32. ``scale``, 0 or more, is 1 / sqrt(head_dim) unless given. A
    node with nothing to see gets zeros."""
    dev = _inputs(q, k_cache, v_cache, lengths, masks)
    code = _lib.act_dtype(q)
    if q.dim() != 4:
        raise ValueError(f"q must be [batch, n, heads, head_dim], got {list(q.shape)}")
    batch, n, heads, dim = q.shape
    _nodes(n)
    shape, ks, vs = _caches(k_cache, v_cache, q.dtype)
    if shape[0] != batch or shape[3] != dim or shape[1] < 1 or heads % shape[1]:
        raise ValueError(f"queries {list(q.shape)} do not fit caches {list(shape)}")
    masks, m_b = _per_node(masks, batch, n, "masks")
    lengths = _int64(lengths, (batch,), "lengths")
    qs = q.stride()
    if qs[3] != 1 or qs[2] != dim or qs[0] % 8 or qs[1] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        qs = q.stride()
    out = torch.empty(batch, n, heads, dim, dtype=q.dtype, device=dev)
    if not batch:
        return out
    ws_bytes = _lib.workspace_size("pe_tree_attention_workspace_size", batch, n, heads, shape[1],
                                   dim, shape[2])
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _call("pe_tree_attention", dev, q.data_ptr(), code, qs[0], qs[1], k_cache.data_ptr(), *ks,
          v_cache.data_ptr(), *vs[:3], lengths.data_ptr(), masks.data_ptr(), m_b, out.data_ptr(),
          batch, n, heads, shape[1], dim, shape[2], 1.0 / math.sqrt(dim) if scale is None else
          scale, _lib.ptr(ws), ws_bytes)
    return out


_LOGIT_DTYPES = {torch.float32: _lib.PE_DTYPE_F32, torch.float16: _lib.PE_DTYPE_F16,
                 torch.bfloat16: _lib.PE_DTYPE_BF16}


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor,
                  parents: Optional[torch.Tensor] = None,
                  draft_probs: Optional[torch.Tensor] = None,
                  temperature: Union[float, torch.Tensor] = 1.0
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand against the target, and the token after them.

    logits [batch, n, vocab] (fp32, fp16 or bf16) of the target at every node;
    tokens int64 [batch, n], -1 where a node is absent (an absent node 0: an empty
    slot); uniforms float32 [batch, n] in [0, 1): ``uniforms[b, c]`` decides node
    c, ``uniforms[b, 0]`` the next token. parents int64 [batch, n] or [n]; None
    for a chain. draft_probs float32 [batch, n - 1, vocab], for a chain: row i is
    what node i + 1 was drawn from; None for drafts that are no random draws (the
    likeliest tokens, a lookup). temperature: a number or float32 [batch]; 0 (in a
    tensor, NaN or less than 0 too) takes the first largest logit.

    The children of a node are tried in order. With p = softmax(logits /
    temperature) child c of token x is accepted if u_c r < p(x), r being what the
    rejected ones left of p, or, drawn from q, if u_c q(x) < p(x). A rejection
    takes x from p, or leaves max(p - q, 0). At the node where no child is left the
    next token is drawn from what is left of p. Returns int64 (out [batch, n]:
    accepted drafts, then the next token; path [batch, n]: accepted nodes from node
    0 on; count [batch]: how many of each; -1 behind them). With n = 1 it samples.
    A sequence whose last distribution has no finite logit gets -1."""
    dev = _inputs(logits, tokens, uniforms, parents, draft_probs,
                  temperature if isinstance(temperature, torch.Tensor) else None)
    code = _LOGIT_DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if logits.dim() != 3:
        raise ValueError(f"logits must be [batch, n, vocab], got {list(logits.shape)}")
    batch, n, vocab = logits.shape
    _nodes(n)
    tokens = _int64(tokens, (batch, n), "tokens")
    if uniforms.dtype is not torch.float32 or uniforms.shape != (batch, n):
        raise ValueError(f"uniforms must be float32 [{batch}, {n}], got {uniforms.dtype} of "
                         f"{list(uniforms.shape)}")
    uniforms = uniforms.contiguous()
    p_b = q_b = q_n = 0
    if parents is not None:
        if draft_probs is not None:
            raise ValueError("draft_probs go with a chain (parents=None)")
        parents, p_b = _per_node(parents, batch, n, "parents")
    if draft_probs is not None:
        if draft_probs.dtype is not torch.float32 or draft_probs.shape != (batch, n - 1, vocab):
            raise ValueError(f"draft_probs must be float32 [{batch}, {n - 1}, {vocab}], got "
                             f"{draft_probs.dtype} of {list(draft_probs.shape)}")
        if n == 1:
            draft_probs = None
        else:
            if vocab > 1 and draft_probs.stride(2) != 1:
                draft_probs = draft_probs.contiguous()
            q_b, q_n = draft_probs.stride(0), draft_probs.stride(1)
    temps, temp = None, 0.0
    if isinstance(temperature, torch.Tensor):
        if temperature.dtype is not torch.float32 or temperature.shape != (batch,):
            raise ValueError(f"temperature must be a number or float32 [{batch}], got "
                             f"{temperature.dtype} of {list(temperature.shape)}")
        temps = temperature.contiguous()
    else:
        temp = float(temperature)
        if not temp >= 0.0:
            raise ValueError(f"temperature must be 0 or more, got {temp}")
    if vocab > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    out = torch.empty(batch, n, dtype=torch.int64, device=dev)
    path = torch.empty(batch, n, dtype=torch.int64, device=dev)
    count = torch.empty(batch, dtype=torch.int64, device=dev)
    if not batch:
        return out, path, count
    ws_bytes = _lib.workspace_size("pe_verify_drafts_workspace_size", batch, n, vocab)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call("pe_verify_drafts", dev, logits.data_ptr(), code, logits.stride(0), logits.stride(1),
          batch, n, vocab, tokens.data_ptr(), _lib.ptr(parents), p_b, uniforms.data_ptr(),
          _lib.ptr(temps), temp, _lib.ptr(draft_probs), q_b, q_n, out.data_ptr(), path.data_ptr(),
          count.data_ptr(), ws.data_ptr(), ws_bytes)
    return out, path, count


def keep_accepted(k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                  path: torch.Tensor, count: torch.Tensor) -> None:
    """The accepted nodes' keys and values to the front of their step: slot
    ``lengths[b] + j`` takes slot ``lengths[b] + path[b, j]``, j < ``count[b]``, in
    caches [batch, kv_heads, positions, head_dim] or, for all layers at once,
    [layers, batch, kv_heads, positions, head_dim]. The slots behind them keep
    what they hold; adding ``count`` to ``lengths`` is the caller's."""
    dev = _inputs(k_cache, v_cache, lengths, path, count)
    if path.dim() != 2:
        raise ValueError(f"path must be [batch, n], got {list(path.shape)}")
    batch, n = path.shape
    _nodes(n)
    path = _int64(path, (batch, n), "path")
    lengths, count = _int64(lengths, (batch,), "lengths"), _int64(count, (batch,), "count")
    views = []
    for name, cache in (("k_cache", k_cache), ("v_cache", v_cache)):
        _lib.act_dtype(cache)
        _writable(cache, name)
        c = cache.unsqueeze(0) if cache.dim() == 4 else cache
        if c.dim() != 5 or c.shape[1] != batch:
            raise ValueError(f"{name} must be [(layers,) {batch}, kv_heads, positions, head_dim], "
                             f"got {list(cache.shape)}")
        views.append(c)
    _apart(k_cache, v_cache)  # moved twice, rows would end up elsewhere
    args = [(c.data_ptr(), c.shape[0], batch, *c.shape[2:], *_strides(c), lengths.data_ptr(),
             path.data_ptr(), count.data_ptr(), n) for c in views if c.numel()]
    if len(args) == 2:  # the values' layout, without layers to move, before the keys move
        _lib.check(_lib.lib().pe_keep_accepted(args[1][0], 0, *args[1][2:], None), "pe_keep_accepted")
    for a in args:
        _call("pe_keep_accepted", dev, *a)
    _written(k_cache, v_cache)
