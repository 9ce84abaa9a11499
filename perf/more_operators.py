"""Operators of serving over a paged 8-bit cache, and of what a step answers with,
measured through the package's public entry points (``own``) and in their plain
form.

Kinds of case (the ranges that ``draw`` covers):

``plan``      block tables and slot maps of a step from the requests' lengths, and
              the blocks back to the pool; 1..1024 sequences, 1..16384 rows.
``write``     keys and values of 1..8192 rows into blocks of 16..128 positions,
              e4m3 codes with one power of two a block and head.
``attend``    attention of 1..2048 new tokens a sequence over such a cache of
              1..130000 positions, all of it or a sliding window with a few first
              positions; 1..64 sequences of different lengths, some slots of the
              batch empty.
``logprobs``  log probabilities of given tokens, their ranks, the entropy and the
              likeliest alternatives of 1..4096 rows over 1000..200000 tokens.

Sequence b of a batch of B has a length and a number of new tokens that the case
alone gives. Blocks that no sequence owns, and slots behind a sequence's end, hold
NaN codes, as memory that nothing has written may.
"""

import math
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "polarengine-vllm_amd"))

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DEV = "cuda"
MOST = 448.0  # the largest e4m3 value
LEAST_E = -100  # the smallest power of two of a block


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step of 64 users: one token each, some of them at a block's end
        {"name": "plan_decode64", "kind": "plan", "batch": 64, "new": 1, "chunks": 0, "len": 4000,
         "ragged": 0.9, "idle": 3, "block": 16, "rows": 64},
        # a large step: 500 users' tokens beside four prompt chunks of odd sizes
        {"name": "plan_mixed500", "kind": "plan", "batch": 500, "new": 1, "chunks": 4, "len": 8000,
         "ragged": 0.9, "idle": 7, "block": 64, "rows": 8192},
        # a decode step's keys and values of 32 users
        {"name": "write_decode32", "kind": "write", "batch": 32, "new": 1, "kv_heads": 8, "dim": 128,
         "block": 64, "len": 4000, "ragged": 0.9, "dtype": "bf16"},
        # five odd chunks into small blocks of a model with small heads
        {"name": "write_odd", "kind": "write", "batch": 5, "new": 333, "kv_heads": 5, "dim": 64,
         "block": 16, "len": 1000, "ragged": 0.7, "dtype": "fp16"},
        # four prompts of 2048 tokens
        {"name": "write_prompts", "kind": "write", "batch": 4, "new": 2048, "kv_heads": 8, "dim": 128,
         "block": 64, "len": 0, "ragged": 0.0, "dtype": "bf16"},
        # one user, a short conversation: latency counts
        {"name": "attend_one_short", "kind": "attend", "batch": 1, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "block": 64, "len": 777, "ragged": 0.0, "idle": 0, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # a full serving batch, one token each, two slots empty
        {"name": "attend_batch32", "kind": "attend", "batch": 32, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "block": 64, "len": 16000, "ragged": 0.6, "idle": 2, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # streaming: long conversations seen through a window and their first tokens, large heads
        {"name": "attend_window_d256", "kind": "attend", "batch": 16, "new": 1, "heads": 32,
         "kv_heads": 16, "dim": 256, "block": 32, "len": 30000, "ragged": 0.9, "idle": 0,
         "window": 4000, "sinks": 4, "dtype": "fp16"},
        # a prompt's chunk behind a long document
        {"name": "attend_chunk1024", "kind": "attend", "batch": 1, "new": 1024, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 64, "len": 30000, "ragged": 0.0, "idle": 0, "window": 0,
         "sinks": 0, "dtype": "bf16"},
        # one answered token of one user, with twenty alternatives
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 20,
         "filtered": False, "dtype": "fp32"},
        # a serving batch with 16-bit logits of an odd vocabulary, filtered to the likeliest
        {"name": "logprobs_batch48", "kind": "logprobs", "rows": 48, "vocab": 100003, "top": 5,
         "filtered": True, "dtype": "bf16"},
        # a prompt's tokens scored
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2048, "vocab": 151936, "top": 1,
         "filtered": False, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "write", "write", "attend", "attend", "attend", "logprobs", "logprobs"])
    if kind == "plan":
        batch = _log(rng, 1, 1024)
        chunks = rng.randrange(min(4, batch) + 1)
        return {"kind": kind, "batch": batch, "new": rng.choice([1, 1, 5]), "chunks": chunks,
                "len": _log(rng, 1, 30000), "ragged": rng.choice([0.0, 0.5, 0.9]),
                "idle": rng.randrange(3) if batch > 8 else 0, "block": rng.choice([16, 32, 64, 128]),
                "rows": 5 * batch + _log(rng, 1, 8192)}
    if kind == "logprobs":
        vocab = _log(rng, 1000, 200_000)
        rows = max(1, min(_log(rng, 1, 4096), 300_000_000 // vocab))
        return {"kind": kind, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]),
                "filtered": rng.random() < 0.4, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    dim = rng.choice([64, 128, 128, 256])
    c = {"kind": kind, "kv_heads": kv, "dim": dim, "block": rng.choice([16, 32, 64, 128]),
         "dtype": rng.choice(["bf16", "fp16"])}
    if kind == "write":
        batch = _log(rng, 1, 64)
        new = rng.choice([1, _log(rng, 1, 4096)])
        new = max(1, min(new, 8192 * 1024 // (batch * kv * dim)))
        return {**c, "batch": batch, "new": new, "len": _log(rng, 1, 4000),
                "ragged": rng.choice([0.0, 0.5, 0.9])}
    group = rng.choice([1, 2, 3, 4, 4, 7, 8])
    length = min(_log(rng, 1, 130_000), 330_000_000 // (kv * dim))
    new = rng.choice([1, 1, _log(rng, 1, 16), _log(rng, 1, 2048)])
    most = min(128_000_000_000 // (kv * group * dim * (length + new)), 340_000_000 // (kv * dim * (length + new)))
    batch = max(1, min(_log(rng, 1, 64), most // new))
    if batch == 1:
        new = max(1, min(new, most))
    return {**c, "batch": batch, "new": new, "heads": kv * group, "len": length,
            "ragged": rng.choice([0.0, 0.3, 0.9]), "idle": rng.choice([0, 1]) if batch > 3 else 0,
            "window": rng.choice([0, 0, _log(rng, 16, 8192)]), "sinks": rng.choice([0, 1, 4, 100])}


def _lengths(case):
    """Cached positions of each sequence, from the case alone: spread down from ``len``
    by up to ``ragged`` of it; -1 marks the ``idle`` empty slots."""
    full, ragged = case["len"], case["ragged"]
    got = [full - int(full * ragged * (b * 0.618 % 1.0)) for b in range(case["batch"])]
    for k in range(case.get("idle", 0)):
        got[1 + 2 * k] = -1
    return got


def _counts(case):
    """New tokens of each sequence: ``new``, fewer for some where it is a chunk's; for a
    plan's ``chunks`` last sequences what is left of the rows, unequal parts of it."""
    got = [case["new"] - int(0.4 * case["new"] * (b * 0.382 % 1.0)) for b in range(case["batch"])]
    got = [0 if n < 0 else c for n, c in zip(_lengths(case), got)]
    chunks = case.get("chunks", 0)
    left = case.get("rows", 0) - sum(got[:len(got) - chunks])
    for k in range(chunks):
        got[len(got) - 1 - k] = max(1, left * (k + 1) * 2 // (chunks * (chunks + 1) + 2))
    return got


def _rows(case):
    return sum(_counts(case))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _tables(case, rng, with_new):
    """Blocks of each sequence for its cached positions (and its new ones), in no order,
    and the other blocks of the pool."""
    t = case["block"]
    most = max(1, max((max(n, 0) + c + t - 1) // t for n, c in zip(_lengths(case), _counts(case))))
    have = [-(-(max(n, 0) + (c if with_new else 0)) // t) for n, c in zip(_lengths(case), _counts(case))]
    spare = 8 + (0 if with_new else sum(c // t + 2 for c in _counts(case)))
    total = sum(have) + spare
    order = np.random.RandomState(rng.randrange(1 << 31)).permutation(total).astype(np.int32)
    tables = np.full((case["batch"], most + 2), -1, np.int32)
    at = 0
    for b, n in enumerate(have):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, order[at:], total


def _codes(shape, g):
    """e4m3 codes of a block whose largest value is near the top of their range."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32 if math.prod(shape) < 1 << 24
                    else torch.bfloat16)
    return x.mul_(75.0).clamp_(-MOST, MOST).to(F8)


def _cache(case, g, tables, total):
    """A cache whose sequences are filled up to their lengths: real codes there, NaN
    codes elsewhere."""
    kv, t, d = case["kv_heads"], case["block"], case["dim"]
    k, v = _codes((total, kv, t, d), g), _codes((total, kv, d, t), g)
    ends = [max(n, 0) + (c if case["kind"] == "attend" else 0)
            for n, c in zip(_lengths(case), _counts(case))]
    used = torch.zeros(total, dtype=torch.int64, device=DEV)  # filled slots of each block
    for b, n in enumerate(ends):
        if n:
            ids = torch.from_numpy(tables[b, :-(-n // t)].astype(np.int64)).to(DEV)
            used[ids] = t
            used[ids[-1:]] = n - (n - 1) // t * t
    empty = torch.arange(t, device=DEV) >= used[:, None]  # [blocks, T]
    k.view(torch.uint8).masked_fill_(empty[:, None, :, None], 0x7F)
    v.view(torch.uint8).masked_fill_(empty[:, None, None, :], 0x7F)
    scales = [torch.randint(127 - 8, 127 - 4, (total, kv), generator=g, device=DEV).to(torch.uint8).view(E8)
              for _ in range(2)]
    return k, v, scales[0], scales[1]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    kind, s = case["kind"], {"case": dict(case)}
    if kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device=DEV).mul_(2.0)
        likely = torch.randint(0, vocab, (rows, 12), generator=g, device=DEV)
        x.scatter_(-1, likely, 8 + 9 * torch.rand(rows, 12, generator=g, device=DEV))
        if case["filtered"]:  # the likeliest tokens alone, as top-k sampling leaves them
            least = x.topk(min(50, vocab), -1).values[:, -1:]
            x.masked_fill_(x < least, -math.inf)
        # most answered tokens are likely ones, some any, a few rows have none
        tokens = likely[torch.arange(rows, device=DEV), torch.randint(0, 12, (rows,), generator=g, device=DEV)]
        other = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        pick = torch.rand(rows, generator=g, device=DEV)
        tokens = torch.where(pick < 0.8, tokens, other)
        tokens = torch.where(pick > 0.98, -1, tokens)
        return {**s, "logits": x.to(DTYPES[case["dtype"]]), "tokens": tokens}
    lengths, counts = _lengths(case), _counts(case)
    s["lengths"] = torch.tensor(lengths, device=DEV)
    s["counts"] = torch.tensor(counts, device=DEV)
    tables, spare, total = _tables(case, rng, kind == "attend")
    if kind == "plan":
        s["tables"] = torch.from_numpy(tables).to(DEV)
        s["free"] = torch.zeros(total, dtype=torch.int32, device=DEV)
        s["free"][:len(spare)] = torch.from_numpy(spare).to(DEV)
        s["free_count"] = torch.tensor([len(spare)], device=DEV)
        return s
    rows, kv, d, dt = sum(counts), case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    s["cache"] = _cache(case, g, tables, total)
    if kind == "attend":
        s["q"] = (torch.randn(rows, case["heads"], d, generator=g, device=DEV) * 1.5).to(dt)
        s["starts"] = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)).to(DEV)
        s["ends"] = torch.where(s["lengths"] < 0, -1, s["lengths"] + s["counts"])
        s["tables"] = torch.from_numpy(tables).to(DEV)
        return s
    # rows to write: their slots, the blocks that the step takes among them
    t, slots = case["block"], []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        have = -(-n // t)
        need = -(-(n + c) // t) - have
        tables[b, have:have + need], spare = spare[:need], spare[need:]
        at = np.arange(n, n + c)
        slots.append(tables[b, at // t].astype(np.int64) * t + at % t)
    s["slots"] = torch.from_numpy(np.concatenate(slots)).to(DEV)
    s["first"] = torch.tensor(np.cumsum([0] + counts[:-1]), device=DEV)
    qkv = torch.randn(rows, 3 * kv, d, generator=g, device=DEV)
    # a token in twenty is an outlier, so that some blocks' scales grow
    qkv *= torch.where(torch.rand(rows, 1, 1, generator=g, device=DEV) < 0.05, 12.0, 1.0)
    qkv = qkv.to(dt)
    s["k"], s["v"] = qkv[:, kv:2 * kv], qkv[:, 2 * kv:]  # views of the projection's rows
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_plan(s):
    c, lengths, counts, tables, free, free_count = s["case"], *(s[k] for k in (
        "lengths", "counts", "tables", "free", "free_count"))
    t, rows, (batch, width) = c["block"], c["rows"], tables.shape
    live = lengths >= 0
    n = torch.where(live, counts.clamp(min=0), 0)
    ends = n.cumsum(0)
    first = ends - n
    j = torch.arange(width, device=tables.device)
    inside = (j >= (lengths // t)[:, None]) & (j <= ((lengths + n - 1) // t)[:, None]) & (n > 0)[:, None]
    fits = live & (lengths + n <= width * t) & (ends <= rows)
    lacks = inside & (tables < 0) & fits[:, None]
    need = lacks.sum(1)
    taken = fits & ((need == 0) | (need.cumsum(0) <= free_count))
    lacks &= taken[:, None]
    rank = lacks.reshape(-1).cumsum(0).view(batch, width) - 1
    got = free[(free_count - 1 - rank).clamp(0, free.numel() - 1)]
    tables.copy_(torch.where(lacks, got, tables))
    free_count -= lacks.sum()
    row = torch.arange(rows, device=tables.device)
    b = torch.searchsorted(ends, row, right=True).clamp(max=batch - 1)
    pos = lengths[b] + row - first[b]
    there = (row < ends[-1]) & taken[b]
    block = tables[b, (pos // t).clamp(0, width - 1)].long()
    return (torch.cat([torch.zeros_like(ends[:1]), ends]).clamp(max=rows), torch.where(there, pos, -1),
            torch.where(there, block * t + pos % t, -1), torch.where(taken, lengths + n, -1))


def _plain_release(s):
    t, tables, free, free_count = s["case"]["block"], s["tables"], s["free"], s["free_count"]
    j = torch.arange(tables.shape[1], device=tables.device)
    back = (j >= ((s["lengths"] + t - 1) // t)[:, None]) & (s["lengths"] >= 0)[:, None] & (tables >= 0)
    total = back.sum()
    rank = back.reshape(-1).cumsum(0).view(back.shape) - 1
    # blocks that stay go to a place behind the stack's end
    at = torch.where(back, free_count + total - 1 - rank, free.numel())
    grown = torch.cat([free, free[:1]])
    free.copy_(grown.scatter(0, at.reshape(-1), tables.reshape(-1))[:-1])
    tables.masked_fill_(back, -1)
    free_count += total


def _power(amax):
    """The smallest e with amax <= 448 2^e, at least LEAST_E."""
    frac, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (frac > 0.875), LEAST_E).clamp(min=LEAST_E)


def _plain_write(codes, scale, x, slots, first, t, by_dim):
    """x [rows, kv_heads, dim] into codes [blocks, kv_heads, T, dim] (or [.., dim, T]);
    first: each sequence's first row, whose block may hold older codes."""
    block, off = slots // t, slots % t
    amax = torch.where(x.isfinite(), x.float().abs(), 0.0).amax(-1)  # [rows, kv_heads]
    exps = scale.view(torch.uint8)
    old = exps.int() - 127
    touched, fresh = torch.zeros(2, old.shape[0], dtype=torch.int32, device=x.device)
    touched[block] = 1
    fresh.scatter_reduce_(0, block, (off == 0).int(), "amax")
    need = torch.full_like(old, LEAST_E)
    need.scatter_reduce_(0, block[:, None].expand_as(amax), _power(amax).int(), "amax")
    need = torch.maximum(need, torch.where(fresh[:, None] == 1, LEAST_E, old))
    new = torch.where(touched[:, None] == 1, need, old)
    ids = block[first]
    shift = torch.where(fresh[:, None] == 1, 0, old - new)[ids]
    by = codes.view(torch.uint8)
    by[ids] = torch.ldexp(codes[ids].float(), shift[..., None, None]).to(F8).view(torch.uint8)
    exps.copy_(new + 127)
    q = torch.ldexp(x.float(), -new[block][..., None])
    q = torch.where(q.isfinite(), q, math.nan).to(F8).view(torch.uint8)
    (by.transpose(-1, -2) if by_dim else by)[block, :, off] = q


def _plain_attend(s):
    c, (kc, vc, ks, vs), tables = s["case"], s["cache"], s["tables"]
    t, kv, d, h = c["block"], c["kv_heads"], c["dim"], c["heads"]
    batch, most, group = c["batch"], max(_counts(c)), h // kv
    last = max(max(n, 0) + m for n, m in zip(_lengths(c), _counts(c)))
    blocks = -(-last // t)
    ids = tables[:, :blocks].long().clamp(min=0)
    k = kc[ids].float() * torch.exp2(ks.view(torch.uint8)[ids].float() - 127)[..., None, None]
    v = vc[ids].float() * torch.exp2(vs.view(torch.uint8)[ids].float() - 127)[..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(batch, kv, blocks * t, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(batch, kv, blocks * t, d)
    pos = torch.arange(blocks * t, device=k.device)
    written = (pos < s["ends"][:, None])[:, None, :, None]
    k, v = k.masked_fill_(~written, 0.0), v.masked_fill_(~written, 0.0)
    i = torch.arange(most, device=k.device)
    row = s["starts"][:-1, None] + i
    there = row < s["starts"][1:, None]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].float()  # [B, most, H, D]
    q = q.view(batch, most, kv, group, d).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, d)
    p = (s["lengths"][:, None] + i)[..., None]  # the new tokens' positions
    seen = (pos <= p) & there[..., None] & (s["ends"] >= 0)[:, None, None]
    if c["window"]:
        seen &= (pos > p - c["window"]) | (pos < c["sinks"])
    sc = torch.matmul(q, k.transpose(-1, -2)).view(batch, kv, most, group, -1).div_(math.sqrt(d))
    sc.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc = sc.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(batch, kv, -1, blocks * t), v).view(batch, kv, most, group, d)
    o = torch.where(total > 0, o / total.clamp(min=1e-30), 0.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(batch, most, h, d).to(s["q"].dtype)
    rows = s["q"].shape[0]
    out = torch.zeros(rows + 1, h, d, dtype=o.dtype, device=o.device)
    out[torch.where(there, row, rows)] = o  # absent rows go to the one behind the last
    return out[:rows]


def _plain_logprobs(s):
    x, tok, top = s["logits"].float() + 0.0, s["tokens"], s["case"]["top"]
    vocab = x.shape[1]
    there = (tok >= 0) & (tok < vocab)
    at = tok.clamp(0, vocab - 1)[:, None]
    best = x.amax(-1, keepdim=True)
    less = x - best
    e = less.exp()
    z = e.sum(-1, dtype=torch.float64)
    entropy = z.log() - torch.where(e > 0, e * less, 0.0).sum(-1, dtype=torch.float64) / z
    xt = x.gather(1, at)
    i = torch.arange(vocab, device=x.device)
    rank = ((x > xt) | ((x == xt) & (i < at))).sum(-1)
    logprob = (xt - best)[:, 0].double() - z.log()
    bits = x.view(torch.int32)
    keys = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 18) + ((1 << 18) - 1 - i)
    key = keys.topk(top, -1).values
    ids = (1 << 18) - 1 - (key & ((1 << 18) - 1))
    alternatives = (x.gather(1, ids) - best).double() - z.log()[:, None]
    return (torch.where(there, logprob, 0.0).float(), torch.where(there, rank, -1), entropy.float(),
            alternatives.float(), ids)


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from polarengine_vllm.kernels import logprobs, paged_cache as pc
    if kind == "logprobs":
        if own:
            return tuple(logprobs.token_logprobs(s["logits"], s["tokens"], c["top"]))
        return _plain_logprobs(s)
    if kind == "plan":
        # the step's blocks go back after it, as when it is called off, so that every
        # pass finds the same pool
        pool = s["tables"], s["free"], s["free_count"]
        if own:
            plan = pc.plan_step(s["lengths"], s["counts"], *pool, c["rows"], c["block"])
            pc.release_blocks(s["tables"], s["lengths"], s["free"], s["free_count"], c["block"])
        else:
            plan = _plain_plan(s)
            _plain_release(s)
        return (*plan, *pool)
    if kind == "write":
        if own:
            pc.write_blocks(s["k"], s["v"], pc.PagedCache(*s["cache"]), s["slots"])
        else:
            k, v, ks, vs = s["cache"]
            _plain_write(k, ks, s["k"], s["slots"], s["first"], c["block"], False)
            _plain_write(v, vs, s["v"], s["slots"], s["first"], c["block"], True)
        return (*s["cache"][:2], *(x.view(torch.uint8) for x in s["cache"][2:]))
    if own:
        return pc.paged_attention(s["q"], pc.PagedCache(*s["cache"]), s["tables"], s["starts"], s["ends"],
                                  window=c["window"] or None, sinks=c["sinks"])
    return _plain_attend(s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _seen(case, length, new):
    """Cached and new positions that at least one of the new tokens sees, and the pairs
    of a new token and a position that it sees."""
    w, s = case["window"] or 1 << 60, case["sinks"] if case["window"] else 0
    low = max(0, length - w + 1)
    positions = length + new - low + min(s, low)
    p = np.arange(length, length + new, dtype=np.float64)
    first = np.maximum(0, p - w + 1)
    return positions, float((p + 1 - first + np.minimum(s, first)).sum())


def work(case):
    kind = case["kind"]
    if kind == "plan":
        taken = sum(c // case["block"] + 1 for c in _counts(case) if c)
        return {"bytes": case["batch"] * 40.0 + case["rows"] * 16.0 + taken * 16.0, "flops": 0.0}
    if kind == "logprobs":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * (4.0 if case["dtype"] == "fp32" else 2.0) + case["rows"] * (28 + 12 * case["top"]),
                "flops": values * 6.0}
    kv, d = case["kv_heads"], case["dim"]
    if kind == "write":
        values = _rows(case) * kv * d * 2.0
        return {"bytes": values * 3 + _rows(case) * 8, "flops": values * 2}
    got = {"bytes": _rows(case) * case["heads"] * d * 4.0, "flops": 0.0}
    for length, new in zip(_lengths(case), _counts(case)):
        if new:
            positions, pairs = _seen(case, length, new)
            got["bytes"] += positions * kv * d * 2.0
            got["flops"] += 4.0 * d * case["heads"] * pairs
    return got


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_plan(s):
    """Sequence by sequence, on the host; the blocks go back in the opposite order."""
    c = s["case"]
    t, rows = c["block"], c["rows"]
    tables, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy().copy()
    count = int(s["free_count"][0])
    starts, pos, slots, ends = [0], np.full(rows, -1), np.full(rows, -1), []
    wanted = taken = 0  # blocks that the sequences so far ask for, and get
    given = []
    for b, (n, m) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
        m = max(m, 0) if n >= 0 else 0
        first = starts[-1]
        starts.append(first + m)
        ok = n >= 0 and n + m <= tables.shape[1] * t and first + m <= rows
        places = [j for j in range(n // t, (n + m - 1) // t + 1) if tables[b, j] < 0] if ok and m else []
        wanted += len(places)
        ok = ok and (not places or wanted <= count)
        ends.append(n + m if ok else -1)
        if not ok:
            continue
        for j in places:
            tables[b, j] = free[count - 1 - taken]
            given.append((b, j))
            taken += 1
        for i in range(m):
            p = n + i
            pos[first + i] = p
            slots[first + i] = int(tables[b, p // t]) * t + p % t
    count -= taken
    for b, j in reversed(given):
        free[count] = tables[b, j]
        tables[b, j] = -1
        count += 1
    whole = lambda a: torch.from_numpy(np.asarray(a, np.int64))  # noqa: E731
    return (whole(np.minimum(starts, rows)), whole(pos), whole(slots), whole(ends),
            torch.from_numpy(tables), torch.from_numpy(free), whole([count]))


def _grid(x):
    """e4m3 values nearest to x (|x| <= 448), ties to even, in 64 bits."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -60))).clamp(min=-6)
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, e)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_write(codes, scale, x, slots, t, by_dim):
    value = codes.double()
    value = value.transpose(-1, -2).contiguous() if by_dim else value
    exps = scale.view(torch.uint8).long()
    at = slots.tolist()
    i = 0
    while i < len(at):
        n = 1
        while i + n < len(at) and at[i + n] == at[i] + n and at[i + n] // t == at[i] // t:
            n += 1
        block, off = at[i] // t, at[i] % t
        rows = x[i:i + n].double().transpose(0, 1)  # [kv_heads, n, dim]
        big = rows.abs().amax((1, 2))
        old = torch.full_like(exps[block], LEAST_E) if off == 0 else exps[block] - 127
        e = torch.ceil(torch.log2(big.clamp(min=2.0 ** -200) / MOST)).long()
        e = torch.where(big <= MOST * torch.exp2(e.double() - 1), e - 1, e)
        e = torch.where(big > MOST * torch.exp2(e.double()), e + 1, e)
        e = torch.maximum(e.clamp(min=LEAST_E), old)
        if off:
            value[block] = _grid(value[block] * torch.exp2((old - e).double())[:, None, None])
        value[block][:, off:off + n] = _grid(rows * torch.exp2(-e.double())[:, None, None])
        exps[block] = e + 127
        i += n
    return value.transpose(-1, -2).contiguous() if by_dim else value, exps.to(torch.uint8)


def _exact_attend(s):
    """One sequence at a time, its new tokens in slices, over the positions that it has."""
    c, (kc, vc, ks, vs), tables = s["case"], s["cache"], s["tables"]
    t, d, h, kv = c["block"], c["dim"], c["heads"], c["kv_heads"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    starts = s["starts"].tolist()
    for b, end in enumerate(s["ends"].tolist()):
        n = starts[b + 1] - starts[b]
        if end < 0 or not n:
            continue
        ids = tables[b, :-(-end // t)].long()
        k = kc[ids].double() * torch.pow(2.0, ks.view(torch.uint8)[ids].double() - 127)[..., None, None]
        v = vc[ids].double() * torch.pow(2.0, vs.view(torch.uint8)[ids].double() - 127)[..., None, None]
        k = k.transpose(1, 2).reshape(-1, kv, d)[:end].permute(1, 2, 0)      # [kv, D, L]
        v = v.permute(0, 3, 1, 2).reshape(-1, kv, d)[:end].transpose(0, 1)   # [kv, L, D]
        j = torch.arange(end, device=q.device)
        step = max(1, (1 << 27) // (h * end))
        for lo in range(0, n, step):
            hi = min(n, lo + step)
            p = torch.arange(end - n + lo, end - n + hi, device=q.device)[:, None]
            hidden = j > p
            if c["window"]:
                hidden |= (j <= p - c["window"]) & (j >= c["sinks"])
            x = q[starts[b] + lo:starts[b] + hi].view(hi - lo, kv, h // kv, d).permute(1, 2, 0, 3)
            w = (x.reshape(kv, -1, d) @ k).view(kv, h // kv, hi - lo, end) / math.sqrt(d)
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            o = (w.view(kv, -1, end) @ v).view(kv, h // kv, hi - lo, d)
            out[starts[b] + lo:starts[b] + hi] = o.permute(2, 0, 1, 3).reshape(hi - lo, h, d)
    return out


def _exact_logprobs(s):
    logits, tokens, top = s["logits"], s["tokens"], s["case"]["top"]
    parts = []
    for r in range(0, logits.shape[0], 256):
        x, tok = logits[r:r + 256].double(), tokens[r:r + 256]
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
        mine = lp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
        xt = x.gather(1, tok.clamp(min=0)[:, None])
        before = (x > xt).sum(-1)
        before += ((x == xt).cumsum(-1).gather(1, tok.clamp(min=0)[:, None]) - 1)[:, 0]
        ids = x.sort(stable=True, dim=-1, descending=True).indices[:, :top]
        parts.append((torch.where(tok >= 0, mine, 0.0), torch.where(tok >= 0, before, -1), entropy,
                      lp.gather(1, ids), ids))
    return tuple(torch.cat(p) for p in zip(*parts))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return _exact_plan(s)
    if kind == "logprobs":
        return _exact_logprobs(s)
    if kind == "attend":
        return _exact_attend(s)
    k, v, ks, vs = s["cache"]
    k, ks = _exact_write(k, ks, s["k"], s["slots"], case["block"], False)
    v, vs = _exact_write(v, vs, s["v"], s["slots"], case["block"], True)
    return k, v, ks, vs
