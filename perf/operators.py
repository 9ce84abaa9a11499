"""Operators of speculative decoding over the decode step's cache, measured
through the package's public entry points (``own``) and in their plain form.

Kinds of case (the ranges that ``draw`` covers):

``rope``    per-head RMS norm of queries and keys with the rotary embedding in
            the same pass, 1..8192 rows; with a cache, keys and values go to
            their slots of it too.
``attend``  attention of 1..64 drafted tokens (a chain or a tree) per sequence
            over a cache of 1..40000 positions; 1..32 sequences of different
            lengths, some slots of the batch empty; keys stored by position
            ("row") or by dimension ("col", the decode runner's layout).
``verify``  which drafted tokens stand against the target's logits, and the
            token that follows them; vocabularies of 1000..200000, greedy and
            sampled, chains with the draft's probabilities and trees without.
``round``   a whole round of a few layers: plan of the trees, norm + rotary +
            cache write, attention, verification, and the accepted tokens' rows
            moved to their places in every layer's cache.

Sequence b of a batch of B has a length that the case alone gives.
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
EPS = 1e-6
DEV = "cuda"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the tree of one user's step, written to the decode runner's cache
        {"name": "rope_tree16", "kind": "rope", "batch": 1, "n": 16, "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "cap": 1100, "len": 1024, "layout": "col", "norm": True,
         "cache": True, "dtype": "bf16"},
        # odd rows of a model whose rotary covers half of a small head, no norms, no cache
        {"name": "rope_odd_half", "kind": "rope", "batch": 1, "n": 1237, "heads": 20, "kv_heads": 5,
         "dim": 64, "rot": 32, "cap": 4096, "len": 0, "layout": "row", "norm": False,
         "cache": False, "dtype": "fp16"},
        # four prompts of 2048 tokens taken into a cache
        {"name": "rope_prefill", "kind": "rope", "batch": 4, "n": 2048, "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "cap": 2304, "len": 130, "layout": "col", "norm": True,
         "cache": True, "dtype": "bf16"},
        # one user, a chain of three drafted tokens, a short conversation: latency counts
        {"name": "attend_chain4_short", "kind": "attend", "batch": 1, "n": 4, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 1100, "len": 777, "ragged": 0.0, "idle": 0,
         "tree": False, "layout": "col", "dtype": "bf16"},
        # a few users of a model with large heads, trees of odd size
        {"name": "attend_tree25_d256", "kind": "attend", "batch": 5, "n": 25, "heads": 32,
         "kv_heads": 16, "dim": 256, "cap": 8192, "len": 8000, "ragged": 0.7, "idle": 1,
         "tree": True, "layout": "row", "dtype": "fp16"},
        # one user with a long document and the largest tree
        {"name": "attend_tree64_long", "kind": "attend", "batch": 1, "n": 64, "heads": 64,
         "kv_heads": 8, "dim": 128, "cap": 33000, "len": 32700, "ragged": 0.0, "idle": 0,
         "tree": True, "layout": "row", "dtype": "bf16"},
        # a full serving batch, chains of seven drafted tokens
        {"name": "attend_batch32", "kind": "attend", "batch": 32, "n": 8, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 16384, "len": 16000, "ragged": 0.6, "idle": 2,
         "tree": False, "layout": "col", "dtype": "bf16"},
        # one user, a chain of four drafted tokens with the draft's probabilities
        {"name": "verify_chain5", "kind": "verify", "batch": 1, "n": 5, "vocab": 151936,
         "tree": False, "temp": "one", "filtered": False, "short": False, "dtype": "fp32"},
        # eight users, the largest trees
        {"name": "verify_tree64", "kind": "verify", "batch": 8, "n": 64, "vocab": 151936,
         "tree": True, "temp": "mixed", "filtered": False, "short": True, "dtype": "fp32"},
        # a serving batch of chains of different lengths, an odd vocabulary, filtered 16-bit logits
        {"name": "verify_chain8_odd", "kind": "verify", "batch": 32, "n": 8, "vocab": 100003,
         "tree": False, "temp": "mixed", "filtered": True, "short": True, "dtype": "bf16"},
        # a whole round of one user's step
        {"name": "round_tree16", "kind": "round", "layers": 4, "batch": 1, "n": 16, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 1100, "len": 1024, "ragged": 0.0, "layout": "col",
         "vocab": 151936, "dtype": "bf16"},
        # a whole round of eight users
        {"name": "round_tree32_b8", "kind": "round", "layers": 2, "batch": 8, "n": 32, "heads": 32,
         "kv_heads": 8, "dim": 128, "cap": 4096, "len": 4000, "ragged": 0.5, "layout": "row",
         "vocab": 151936, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "attend", "attend", "verify", "verify", "round"])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8])
    dim = rng.choice([64, 128, 128, 256])
    c = {"kind": kind, "layout": rng.choice(["row", "col"]), "dtype": rng.choice(["bf16", "fp16"])}
    if kind == "rope":
        batch = _log(rng, 1, 16)
        n = max(1, min(_log(rng, 1, 4096), 50_000_000 // (batch * kv * (group + 2) * dim)))
        start = _log(rng, 1, 4000)
        return {**c, "batch": batch, "n": n, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "cap": start + n + rng.randrange(300),
                "len": start, "norm": rng.random() < 0.7, "cache": rng.random() < 0.7}
    if kind == "attend":
        n = _log(rng, 1, 64)
        length = _log(rng, 1, 40000)
        most = min(130_000_000 // (kv * group * n * length), 800_000_000 // (kv * dim * length))
        batch = max(1, min(_log(rng, 1, 32), most))
        if batch == 1:  # one long sequence: its tree and heads within the largest case's work
            n = max(1, min(n, 130_000_000 // (kv * group * length)))
        return {**c, "batch": batch, "n": n, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "cap": length + n + rng.randrange(300), "len": length,
                "ragged": rng.choice([0.0, 0.3, 0.9]), "idle": rng.choice([0, 1]) if batch > 3 else 0,
                "tree": rng.random() < 0.6}
    vocab = _log(rng, 1000, 200_000)
    n = _log(rng, 1, 64)
    batch = max(1, min(_log(rng, 1, 64), 70_000_000 // (vocab * n)))
    if kind == "verify":
        del c["layout"]
        return {**c, "batch": batch, "n": n, "vocab": vocab, "tree": rng.random() < 0.5,
                "temp": rng.choice(["one", "mixed", "greedy"]), "filtered": rng.random() < 0.4,
                "short": rng.random() < 0.5, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    length = _log(rng, 1, 4000)
    batch = min(batch, 8)
    return {**c, "layers": rng.choice([1, 2, 3]), "batch": batch, "n": n, "heads": kv * group,
            "kv_heads": kv, "dim": dim, "cap": length + n + rng.randrange(200), "len": length,
            "ragged": rng.choice([0.0, 0.5]), "vocab": vocab}


def _lengths(case):
    """Length of each sequence, from the case alone: spread down from ``len`` by
    up to ``ragged`` of it; -1 marks the ``idle`` empty slots."""
    full, ragged = case["len"], case.get("ragged", 0.0)
    got = [max(0, full - int(full * ragged * (b * 0.618 % 1.0))) for b in range(case["batch"])]
    for k in range(case.get("idle", 0)):
        got[1 + 2 * k] = -1
    return got


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _trees(rng, case):
    """Parents, one tree per sequence: a chain, or a tree whose nodes hang mostly on
    recent ones, as drafts that expand the likeliest leaves make them."""
    if not case.get("tree", True):
        return [[i - 1 for i in range(case["n"])] for _ in range(case["batch"])]
    return [[-1] + [max(0, i - 1 - int(rng.expovariate(0.25))) for i in range(1, case["n"])]
            for _ in range(case["batch"])]


def _bits(parents):
    masks = []
    for i, p in enumerate(parents):
        masks.append((1 << i) | (masks[p] if i else 0))
    return masks


def _signed(m):
    return m - (1 << 64) if m >> 63 else m


def _rope_table(cap, rot):
    inv = 1.0e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    ang = torch.arange(cap, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _caches(case, g, layers, dt):
    """K and V [layers, batch, kv_heads, cap, dim]; "col": K stored by dimension."""
    shape = [layers, case["batch"], case["kv_heads"], case["cap"], case["dim"]]
    col = shape[:3] + [shape[4], shape[3]]
    k = torch.randn(col if case["layout"] == "col" else shape, generator=g, device=DEV, dtype=dt)
    v = torch.randn(shape, generator=g, device=DEV, dtype=dt)
    return k.transpose(-1, -2) if case["layout"] == "col" else k, v


def _drafts(case, g, rng, parents):
    """Logits of the target for every node (a wide floor and a few likely tokens),
    drafted tokens and what verification takes beside them. A draft agrees with the target up to noise: a chain's tokens
    are drawn from its probabilities, a tree's are its likeliest at each node."""
    b, n, vocab = case["batch"], case["n"], case["vocab"]
    dt = DTYPES[case["dtype"]] if case["kind"] == "verify" else torch.float32
    x = torch.randn(b, n, vocab, generator=g, device=DEV) * 2.0
    likely = torch.randint(0, vocab, (b, n, 12), generator=g, device=DEV)
    x.scatter_(-1, likely, 8 + 9 * torch.rand(b, n, 12, generator=g, device=DEV))
    if case.get("filtered"):  # the likeliest tokens alone, as top-k sampling leaves them
        least = x.topk(min(50, vocab), -1).values[..., -1:]
        x = x.masked_fill(x < least, -math.inf)
    logits = x.to(dt)
    guess = x + 0.6 * torch.randn(b, n, vocab, generator=g, device=DEV)
    par = torch.tensor(parents, device=DEV)
    tokens = torch.zeros(b, n, dtype=torch.int64, device=DEV)
    probs = None
    if case.get("tree", True):
        most = max(tree[1:].count(p) for tree in parents for p in tree) if n > 1 else 1
        rank = torch.tensor([[tree[1:i].count(p) if i else 0 for i, p in enumerate(tree)]
                             for tree in parents], device=DEV)
        best = guess.topk(min(max(1, most), vocab), -1).indices
        row = best.gather(1, par.clamp(min=0)[..., None].expand(-1, -1, best.shape[2]))
        tokens = row.gather(2, rank.clamp(max=best.shape[2] - 1)[..., None])[..., 0]
    elif n > 1:
        probs = torch.softmax(guess[:, :-1], -1)
        gumbel = -torch.empty_like(probs).exponential_(generator=g).log()
        tokens[:, 1:] = (probs.log() + gumbel).argmax(-1)
    tokens[:, 0] = torch.randint(0, vocab, (b,), generator=g, device=DEV)
    if case.get("short"):  # sequences with fewer drafted tokens than the batch has room for
        for s in range(0, b, 3):
            tokens[s, max(1, n - 1 - s % max(1, n)):] = -1
    u = torch.rand(b, n, generator=g, device=DEV)
    temps = {"one": [1.0], "greedy": [0.0], "mixed": [0.0, 0.6, 1.0, 1.3]}[case.get("temp", "one")]
    temp = torch.tensor([temps[s % len(temps)] for s in range(b)], device=DEV)
    return {"logits": logits, "tokens": tokens, "u": u, "temp": temp, "probs": probs,
            "parents": par if case.get("tree", True) else None}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    kind, s = case["kind"], {"case": dict(case)}
    if kind == "verify":
        return {**s, **_drafts(case, g, rng, _trees(rng, case))}
    b, n, h, kv, d = (case[k] for k in ("batch", "n", "heads", "kv_heads", "dim"))
    dt = DTYPES[case["dtype"]]
    s["lengths"] = torch.tensor(_lengths(case), device=DEV)
    if kind == "attend":
        s["masks"] = torch.tensor([[_signed(m) for m in _bits(t)] for t in _trees(rng, case)],
                                  device=DEV)
        s["q"] = (torch.randn(b, n, h, d, generator=g, device=DEV) * 1.5).to(dt)
        k, v = _caches(case, g, 1, dt)
        return {**s, "k": k[0], "v": v[0]}
    layers = case.get("layers", 1)
    s["qkv"] = [torch.randn(b * n, (h + 2 * kv) * d, generator=g, device=DEV).to(dt)
                for _ in range(layers)]
    s["rope"] = _rope_table(case["cap"], case.get("rot", d))
    s["qw"], s["kw"] = ((1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
                        if case.get("norm", True) else None for _ in range(2))
    if case.get("cache", True):
        s["k"], s["v"] = _caches(case, g, layers, dt)
    if kind == "rope":
        s["positions"] = s["lengths"][:, None] + torch.arange(n, device=DEV)
        return s
    return {**s, **_drafts(case, g, rng, _trees(rng, case))}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_rope(s, qkv, positions):
    """fp32 normed and rotated queries and keys [rows, heads, dim], and the values."""
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    rows = qkv.view(-1, h + 2 * kv, d)
    half = s["rope"].shape[1] // 2
    cos, sin = s["rope"][positions.reshape(-1)][:, None].split(half, -1)

    def one(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1).to(qkv.dtype)

    return one(rows[:, :h], s["qw"]), one(rows[:, h:h + kv], s["kw"]), rows[:, h + kv:]


def _plain_write(cache, rows, lengths):
    """rows [B * n, kv_heads, dim] into the slots from ``lengths`` on."""
    b = cache.shape[0]
    rows = rows.reshape(b, -1, *rows.shape[1:])
    slots = lengths[:, None] + torch.arange(rows.shape[1], device=cache.device)
    cache[torch.arange(b, device=cache.device)[:, None], :, slots] = rows


def _plain_attend(q, k, v, lengths, masks):
    b, n, h, d = q.shape
    kv, cap = k.shape[1], k.shape[2]
    j = torch.arange(cap, device=q.device)
    rel = j - lengths[:, None]  # [B, cap]: a draft's place behind the sequence
    drafted = (masks[..., None] >> rel[:, None].clamp(0, 63)) & 1
    seen = (rel < 0)[:, None] | ((rel >= 0) & (rel < n))[:, None] & (drafted == 1)
    seen &= (lengths >= 0)[:, None, None]
    x = q.float().view(b, n, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    sc = torch.matmul(x, k.float().transpose(-1, -2)).view(b, kv, n, h // kv, cap) / math.sqrt(d)
    sc = sc.masked_fill(~seen[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, kv, -1, cap), v.float()).view(b, kv, n, h // kv, d)
    o = torch.where(total > 0, o / total.clamp(min=1e-30), 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(b, n, h, d).to(q.dtype)


def _plain_tree(parents):
    """[B, N, N]: whether j is i or an ancestor of i (paths of any number of steps)."""
    n = parents.shape[1]
    j = torch.arange(n, device=parents.device)
    step = ((parents[..., None] == j) & (j > 0)[:, None]).double()
    return torch.matrix_power(torch.eye(n, device=parents.device, dtype=torch.float64) + step, 64) > 0


def _plain_verify(s):
    x, tok, u, probs = s["logits"].double(), s["tokens"], s["u"].double(), s["probs"]
    b, n, vocab = x.shape
    dev = x.device
    i = torch.arange(n, device=dev)
    par = s["parents"] if s["parents"] is not None else (i - 1).expand(b, n)
    temp = s["temp"].double()[:, None, None]
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(vocab, device=dev), vocab).amin(-1, keepdim=True)
    w = torch.exp((x - top) / temp.clamp(min=1e-30))
    w = torch.where(temp > 0, w, torch.zeros_like(w).scatter_(-1, first, 1.0))
    p = w / w.sum(-1, keepdim=True)

    there = (tok >= 0) & (par >= 0)  # a drafted token
    at = par.clamp(min=0)[..., None].expand(-1, -1, vocab)
    px = p.gather(1, at).gather(2, tok.clamp(min=0)[..., None])[..., 0]
    sib = (par[:, :, None] == par[:, None]) & (i[None] < i[:, None]) & there[:, None]  # [B, i, earlier j]
    if probs is not None:
        qx = probs.double().gather(2, tok[:, 1:].clamp(min=0)[..., None])[..., 0]
        ok = u * torch.cat([torch.ones_like(qx[:, :1]), qx], 1) < px
    else:
        px = torch.where((sib & (tok[:, :, None] == tok[:, None])).any(-1), 0.0, px)
        ok = u * (1 - (sib * px[:, None]).sum(-1)) < px
    ok &= there
    taken = ok & ~(sib & ok[:, None]).any(-1)
    taken[:, 0] = True
    on = ~(_plain_tree(par) & ~taken[:, None]).any(-1)  # on the accepted path
    count = on.sum(-1)
    last = torch.where(on, i, 0).amax(-1)

    left = p.gather(1, last[:, None, None].expand(-1, 1, vocab))[:, 0]
    child = (par == last[:, None]) & there
    if probs is not None:
        row = last.clamp(max=n - 2)[:, None, None].expand(-1, 1, vocab)
        rest = (left - probs.double().gather(1, row)[:, 0]).clamp(min=0)
        rest = torch.where(child.any(-1, keepdim=True), rest, left)
    else:
        gone = torch.zeros(b, vocab, device=dev).scatter_add_(1, tok.clamp(min=0), child.float())
        rest = torch.where(gone > 0, 0.0, left)
    left = torch.where(rest.sum(-1, keepdim=True) > 0, rest, left)
    cum = left.cumsum(-1)
    new = (cum <= u[:, :1] * cum[:, -1:]).sum(-1).clamp(max=vocab - 1)

    path = torch.where(on, i, n).sort(-1).values
    said = torch.cat([tok, tok[:, :1]], 1).gather(1, path.roll(-1, 1))
    said = torch.where(i == (count - 1)[:, None], new[:, None], said)
    inside = i < count[:, None]
    return torch.where(inside, said, -1), torch.where(inside, path, -1), count


def _plain_keep(cache, lengths, path, count, n):
    """cache [layers, B, kv_heads, cap, dim]: rows of the accepted path to the front."""
    b = cache.shape[1]
    j = torch.arange(n, device=cache.device)
    row = torch.arange(b, device=cache.device)[:, None]
    src = lengths[:, None] + torch.where(j < count[:, None], path, j)
    cache[:, row, :, lengths[:, None] + j] = cache[:, row, :, src]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from polarengine_vllm.kernels import tree_decode as td
    if kind == "attend":
        if own:
            return td.tree_attention(s["q"], s["k"], s["v"], s["lengths"], s["masks"])
        return _plain_attend(s["q"], s["k"], s["v"], s["lengths"], s["masks"])
    if kind == "verify":
        if own:
            return td.verify_drafts(s["logits"], s["tokens"], s["u"], parents=s["parents"],
                                    draft_probs=s["probs"], temperature=s["temp"])
        return _plain_verify(s)
    h, kv = c["heads"], c["kv_heads"]
    if kind == "rope":
        qkv, pos = s["qkv"][0], s["positions"]
        if own and not c["cache"]:
            return td.qk_norm_rope(qkv, h, kv, s["rope"], pos, s["qw"], s["kw"], EPS)
        if own:
            q = td.qk_norm_rope_write(qkv, h, kv, s["rope"], pos, s["k"][0], s["v"][0],
                                      s["lengths"], s["qw"], s["kw"], EPS)
            return q, s["k"][0], s["v"][0]
        q, k, v = _plain_rope(s, qkv, pos)
        if not c["cache"]:
            return q, k
        _plain_write(s["k"][0], k, s["lengths"])
        _plain_write(s["v"][0], v, s["lengths"])
        return q, s["k"][0], s["v"][0]
    # a round
    outs = []
    if own:
        plan = td.tree_plan(s["parents"], s["lengths"])
        for i, qkv in enumerate(s["qkv"]):
            q = td.qk_norm_rope_write(qkv, h, kv, s["rope"], plan.positions, s["k"][i], s["v"][i],
                                      s["lengths"], s["qw"], s["kw"], EPS)
            outs.append(td.tree_attention(q.view(c["batch"], c["n"], h, c["dim"]), s["k"][i],
                                          s["v"][i], s["lengths"], plan.masks))
        tokens, path, count = td.verify_drafts(s["logits"], s["tokens"], s["u"],
                                               parents=s["parents"], temperature=s["temp"])
        td.keep_accepted(s["k"], s["v"], s["lengths"], path, count)
        return outs, tokens, path, count, s["k"], s["v"]
    tree = _plain_tree(s["parents"])
    pos = s["lengths"][:, None] + tree.sum(-1) - 1
    masks = (tree.long() << torch.arange(c["n"], device=DEV)).sum(-1)
    for i, qkv in enumerate(s["qkv"]):
        q, k, v = _plain_rope(s, qkv, pos)
        _plain_write(s["k"][i], k, s["lengths"])
        _plain_write(s["v"][i], v, s["lengths"])
        outs.append(_plain_attend(q.view(c["batch"], c["n"], h, c["dim"]), s["k"][i], s["v"][i],
                                  s["lengths"], masks))
    tokens, path, count = _plain_verify(s)
    _plain_keep(s["k"], s["lengths"], path, count, c["n"])
    _plain_keep(s["v"], s["lengths"], path, count, c["n"])
    return outs, tokens, path, count, s["k"], s["v"]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    got = {"bytes": 0.0, "flops": 0.0}
    if kind in ("rope", "round"):
        rows, layers = case["batch"] * case["n"], case.get("layers", 1)
        heads = case["heads"] + case["kv_heads"] * (2 if case.get("cache", True) else 1)
        got["bytes"] += layers * rows * heads * case["dim"] * 2 * 2
        got["flops"] += layers * rows * (case["heads"] + case["kv_heads"]) * case["dim"] * 7
    if kind in ("attend", "round"):
        layers = case.get("layers", 1)
        seen = sum(v + case["n"] for v in _lengths(case) if v >= 0)
        q = case["batch"] * case["n"] * case["heads"] * case["dim"]
        got["bytes"] += layers * (seen * case["kv_heads"] * case["dim"] * 2 * 2 + q * 2 * 2)
        got["flops"] += layers * 4.0 * case["n"] * case["heads"] * case["dim"] * seen
    if kind in ("verify", "round"):
        size = {"fp32": 4}.get(case["dtype"], 2) if kind == "verify" else 4
        values = case["batch"] * case["n"] * case["vocab"]
        chain = kind == "verify" and not case["tree"] and case["n"] > 1
        got["bytes"] += values * size + (case["batch"] * case["vocab"] * 4 if chain else 0)
        got["flops"] += values * 4.0
    return got


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rope(s, qkv, pos):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    x = qkv.double().view(-1, h + 2 * kv, d)
    r = s["rope"].shape[1]
    ang = s["rope"].double()[pos.reshape(-1)]
    z = torch.complex(ang[:, :r // 2], ang[:, r // 2:])[:, None]  # a rotation is a complex factor

    def one(x, w):
        if w is not None:
            x = x / x.pow(2).mean(-1, keepdim=True).add(EPS).sqrt() * w.double()
        y = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * z
        return torch.cat([y.real, y.imag, x[..., r:]], -1)

    return one(x[:, :h], s["qw"]), one(x[:, h:h + kv], s["kw"]), x[:, h + kv:]


def _exact_attend(q, k, v, lengths, masks):
    """One sequence and one drafted token at a time, over the positions that it sees."""
    b, n, h, d = q.shape
    g = h // k.shape[1]
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device=q.device)
    for s, length in enumerate(lengths.tolist()):
        if length < 0:
            continue
        kd, vd = k[s, :, :length + n].double(), v[s, :, :length + n].double()
        base = torch.arange(length, device=q.device)
        for t, bits in enumerate(masks[s].tolist()):
            draft = [length + j for j in range(n) if bits >> j & 1]
            where = torch.cat([base, torch.tensor(draft, device=q.device, dtype=torch.int64)])
            if not where.numel():
                continue
            kt, vt = kd[:, where], vd[:, where]
            sc = (q[s, t].double().view(-1, g, d) @ kt.transpose(-1, -2)) / math.sqrt(d)
            out[s, t] = (torch.softmax(sc, -1) @ vt).reshape(h, d)
    return out


def _exact_verify(s):
    """The walk from node to node, in numpy."""
    logits, tok, u = s["logits"].float().cpu().numpy(), s["tokens"].tolist(), s["u"].double().tolist()
    temp, probs = s["temp"].tolist(), s["probs"]
    b, n, vocab = logits.shape
    tokens, path = np.full((b, n), -1, np.int64), np.full((b, n), -1, np.int64)
    count = np.zeros(b, np.int64)
    for r in range(b):
        par = s["parents"][r].tolist() if s["parents"] is not None else [i - 1 for i in range(n)]
        node, steps, said = 0, [0], []
        while True:
            x = logits[r, node].astype(np.float64)
            if temp[r] > 0:
                left = np.exp((x - x.max()) / temp[r])
                left /= left.sum()
            else:
                left = (np.arange(vocab) == x.argmax()).astype(np.float64)
            kids = [i for i in range(1, n) if par[i] == node and tok[r][i] >= 0]
            went = None
            for c in kids:
                t = tok[r][c]
                if probs is not None:
                    q = probs[r, node].double().cpu().numpy()
                    if u[r][c] * q[t] < left[t]:
                        went = c
                        break
                    rest = np.maximum(left - q, 0)
                else:
                    if u[r][c] * left.sum() < left[t]:
                        went = c
                        break
                    rest = left.copy()
                    rest[t] = 0
                left = rest if rest.sum() > 0 else left
            if went is None:
                break
            node = went
            steps.append(went)
            said.append(tok[r][went])
        cum = np.cumsum(left)
        said.append(min(int(np.searchsorted(cum, u[r][0] * cum[-1], side="right")), vocab - 1))
        count[r] = len(steps)
        path[r, :len(steps)], tokens[r, :len(said)] = steps, said
    return tuple(torch.from_numpy(a) for a in (tokens, path, count))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend":
        return _exact_attend(s["q"], s["k"], s["v"], s["lengths"], s["masks"])
    if kind == "verify":
        return _exact_verify(s)
    b, n, h = case["batch"], case["n"], case["heads"]
    if kind == "rope":
        q, k, v = _exact_rope(s, s["qkv"][0], s["positions"])
        if not case["cache"]:
            return q, k
        caches = [s["k"][0].double(), s["v"][0].double()]
        for r, start in enumerate(s["lengths"].tolist()):
            for cache, new in zip(caches, (k, v)):
                cache[r, :, start:start + n] = new.view(b, n, *new.shape[1:])[r].transpose(0, 1)
        return q, caches[0], caches[1]
    masks, depth = [], []
    for t in s["parents"].tolist():
        masks.append([_signed(m) for m in _bits(t)])
        depth.append([bin(m).count("1") - 1 for m in _bits(t)])
    pos = s["lengths"][:, None] + torch.tensor(depth, device=DEV)
    masks = torch.tensor(masks, device=DEV)
    tokens, path, count = _exact_verify(s)
    caches, outs = [s["k"].double(), s["v"].double()], []
    for i, qkv in enumerate(s["qkv"]):
        q, k, v = _exact_rope(s, qkv, pos)
        dt = qkv.dtype  # queries and the cache are of this type: what is stored is rounded to it
        for cache, new in zip(caches, (k, v)):
            for r, start in enumerate(s["lengths"].tolist()):
                new_r = new.view(b, n, *new.shape[1:])[r].transpose(0, 1)
                cache[i, r, :, start:start + n] = new_r.to(dt).double()
        outs.append(_exact_attend(q.to(dt).view(b, n, h, -1), caches[0][i], caches[1][i],
                                  s["lengths"], masks))
        for r, start in enumerate(s["lengths"].tolist()):
            kept = [p for p in path[r].tolist() if p >= 0]
            for cache in caches:
                at = torch.tensor([start + p for p in kept], device=DEV)
                cache[i, r][:, start:start + len(kept)] = cache[i, r][:, at]
    return outs, tokens, path, count, caches[0], caches[1]
