"""GPU tests of the kernels for drafted tokens (polarengine_vllm.kernels.tree_decode)
against float64 statements of the same inputs on the CPU.

Tolerances. A result rounded once to 16 bits is off by at most half a step,
h = finfo.eps / 2 of its value (and half the smallest subnormal). Norm and rotation
before it: sums of at most 256 fp32 squares and a handful of fp32 operations, under
2^-18 of the turned pair's size. Attention: each probability is rounded to 16 bits
(h of itself), in the sum of the values and, alike or not, in the sum that divides
them, so the result is off by at most 2 h of A = sum p |v| / sum p; fp32 scores are
off by less than 2^-13 (256 products of size 8 at most), which adds 2^-12 A; an fp16
probability below the normal range adds 2^-25 |v| at most. Verification answers in
whole numbers and has to be equal."""

import math
import random

import numpy as np
import pytest
import torch

from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu

EPS = 1e-6
NAN, INF = float("nan"), float("inf")


def _td():
    from polarengine_vllm.kernels import tree_decode
    return tree_decode


def _tree(rng, n, spread=4):
    return [-1] + [max(0, i - 1 - rng.randrange(spread)) for i in range(1, n)]


def _bits(parents):
    masks = []
    for i, p in enumerate(parents):
        up = 1 if i == 0 else masks[p] if 0 <= p < i else 0
        masks.append(up | 1 << i if i == 0 or up else 0)
    return masks


def _signed(m):
    return m - (1 << 64) if m >> 63 else m


def _i64(x):
    return torch.tensor(x, dtype=torch.int64)


# ---------------------------------------------------------------------------
# tree_plan
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 2, 3, 16, 63, 64])
@pytest.mark.parametrize("shared", [False, True])
def test_plan(n, shared):
    say(f"plan n={n} shared={shared}")
    rng = random.Random(n)
    lengths = [0, 1, 777, -1, 1 << 40]
    trees = [_tree(rng, n, 1 + 3 * b) for b in range(5)]
    if n > 2:
        trees[1][n // 2] = -1           # absent, and what hangs on it
        trees[2][1] = 1                 # its own parent
        trees[4][2], trees[0][0] = n, 5  # a later parent; the root's is not looked at
    if shared:
        trees = trees[:1] * 5
    par = _i64(trees[0] if shared else trees).to(DEV)
    got = _td().tree_plan(par, _i64(lengths).to(DEV))
    masks = [_bits(t) for t in trees]
    want = [[length + bin(m).count("1") - 1 if m and length >= 0 else -1 for m in ms]
            for ms, length in zip(masks, lengths)]
    assert got.positions.tolist() == want
    assert got.masks.tolist() == [[_signed(m) for m in ms] for ms in masks]


# ---------------------------------------------------------------------------
# norm + rotary
# ---------------------------------------------------------------------------
def _rope_ref(qkv, heads, kv, table, pos, qw, kw):
    """float64 queries, keys and the size of each rotated pair."""
    d = qkv.shape[1] // (heads + 2 * kv)
    x = qkv.double().view(qkv.shape[0], -1, d)
    r = table.shape[1]
    ok = (pos >= 0) & (pos < table.shape[0])
    t = table.double()[pos.clamp(0, table.shape[0] - 1)][:, None]
    cos, sin = t[..., :r // 2], t[..., r // 2:]
    out = []
    for y, w in ((x[:, :heads], qw), (x[:, heads:heads + kv], kw)):
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
        a, b = y[..., :r // 2], y[..., r // 2:r]
        z = torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., r:]], -1)
        size = torch.cat([a.abs() + b.abs()] * 2 + [y[..., r:].abs()], -1)
        out.append((torch.where(ok[:, None, None], z, 0.0), size))
    return out


def _close16(got, want, size, what):
    f = torch.finfo(got.dtype)
    err = (got.double().cpu() - want).abs()
    tol = f.eps / 2 * want.abs() + size * 2.0 ** -18 + f.smallest_normal * f.eps / 2
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, worst {float(err[bad].max()):.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,heads,kv,dim,rot", [
    (1, 1, 1, 64, 64), (3, 5, 1, 128, 128), (37, 32, 8, 128, 64), (130, 4, 2, 256, 256),
    (9, 6, 3, 256, 48), (5, 7, 7, 64, 16), (2, 32, 8, 128, 96)])
@pytest.mark.parametrize("norm", ["both", "none", "q"])
def test_norm_rope(dtype, rows, heads, kv, dim, rot, norm):
    say(f"norm_rope {dtype} rows={rows} heads={heads}/{kv} dim={dim} rot={rot} norm={norm}")
    g = torch.Generator().manual_seed(rows * dim + rot)
    qkv = (torch.randn(rows, (heads + 2 * kv) * dim, generator=g) * 3).to(dtype)
    qkv[rows // 2, :dim] = 0
    table = torch.rand(50, rot, generator=g) * 2 - 1
    pos = torch.randint(0, 50, (rows,), generator=g)
    if rows > 2:
        pos[0], pos[1], pos[2] = -1, 50, 49
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2)]
    qw, kw = (w[0] if norm != "none" else None), (w[1] if norm == "both" else None)
    dev = [t if t is None else t.to(DEV) for t in (qkv, table, pos, qw, kw)]
    q, k = _td().qk_norm_rope(dev[0], heads, kv, dev[1], dev[2], dev[3], dev[4], EPS)
    for got, (want, size), what in zip((q, k), _rope_ref(qkv, heads, kv, table, pos, qw, kw), "qk"):
        _close16(got, want, size, what)


@pytest.mark.parametrize("case", ["strided", "unaligned", "empty", "transposed"])
def test_norm_rope_layouts(case):
    say(f"norm_rope layout {case}")
    g = torch.Generator().manual_seed(3)
    rows = 0 if case == "empty" else 6
    base = torch.randn(rows, 8 * 64, generator=g).to(torch.bfloat16).to(DEV)
    table = torch.rand(9, 64, generator=g).to(DEV)
    pos = torch.arange(rows, device=DEV)
    want = _td().qk_norm_rope(base, 4, 2, table, pos)
    if case == "strided":
        qkv = torch.zeros(rows, 8 * 64 + 40, dtype=base.dtype, device=DEV)[:, 24:24 + 512]
    elif case == "unaligned":
        qkv = torch.zeros(rows, 8 * 64 + 3, dtype=base.dtype, device=DEV)[:, 1:513]
    else:
        qkv = torch.zeros(8 * 64, rows, dtype=base.dtype, device=DEV).t()
    qkv.copy_(base)
    got = _td().qk_norm_rope(qkv, 4, 2, table, pos)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def _cache(batch, kv, cap, dim, dtype, layout, fill, g=None, layers=None):
    lead = (batch, kv) if layers is None else (layers, batch, kv)
    shape = lead + ((dim, cap) if layout == "col" else (cap, dim))
    if layout == "gap":  # rows within a wider tensor
        t = torch.full(lead + (cap, dim + 24), fill, dtype=dtype)[..., 8:8 + dim]
    else:
        t = torch.full(shape, fill, dtype=dtype)
    if g is not None:
        t.copy_(torch.randn(t.shape, generator=g).to(dtype))
    dev = torch.empty_strided(t.shape, t.stride(), dtype=dtype, device=DEV)
    dev.copy_(t)
    return dev.transpose(-1, -2) if layout == "col" else dev


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["row", "col", "gap"])
@pytest.mark.parametrize("n,dim", [(1, 128), (5, 64), (64, 128), (130, 128), (33, 256)])
def test_norm_rope_write(dtype, layout, n, dim):
    say(f"norm_rope_write {dtype} {layout} n={n} dim={dim}")
    td, g = _td(), torch.Generator().manual_seed(n + dim)
    heads, kv, cap, lens = 6, 3, n + 21, [0, 21, 22, -1, 7]
    b = len(lens)
    qkv = torch.randn(b * n, (heads + 2 * kv) * dim, generator=g).to(dtype).to(DEV)
    table = torch.rand(cap, dim, generator=g).to(DEV)
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype).to(DEV)
    lengths = _i64(lens)
    pos = (lengths[:, None] + torch.arange(n)).clamp(0, cap - 1)
    pos[4, n // 2] = -1
    k, v = (_cache(b, kv, cap, dim, dtype, y, NAN) for y in (layout, "gap" if layout == "gap" else "row"))
    got = td.qk_norm_rope_write(qkv, heads, kv, table, pos.to(DEV), k, v, lengths.to(DEV), w, w, EPS)
    q, rows = td.qk_norm_rope(qkv, heads, kv, table, pos.to(DEV), w, w, EPS)
    assert torch.equal(got, q)
    vals = qkv.view(b, n, heads + 2 * kv, dim)[:, :, heads + kv:]
    want = [torch.full((b, kv, cap, dim), NAN, dtype=dtype) for _ in range(2)]
    for s, length in enumerate(lens):
        for i in range(n):
            if 0 <= length <= cap - n and pos[s, i] >= 0:
                want[0][s, :, length + i] = rows.view(b, n, kv, dim)[s, i].cpu()
                want[1][s, :, length + i] = vals[s, i].cpu()
    for have, w_ in zip((k, v), want):
        assert torch.equal(have.cpu().contiguous().view(torch.int16), w_.view(torch.int16))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attend_ref(q, k, v, lengths, masks, scale):
    """float64 outputs and A = sum p |v| / sum p, and the sum of |v| seen."""
    b, n, h, d = q.shape
    grp = h // k.shape[1]
    out, size, total = (torch.zeros(b, n, h, d, dtype=torch.float64) for _ in range(3))
    for s in range(b):
        length = int(lengths[s])
        if length < 0 or length > k.shape[2] - n:
            continue
        for i in range(n):
            at = list(range(length)) + [length + j for j in range(n) if int(masks[s, i]) >> j & 1]
            if not at:
                continue
            for x in range(h):
                kk, vv = k[s, x // grp, at].double(), v[s, x // grp, at].double()
                p = torch.softmax(kk @ q[s, i, x].double() * scale, 0)
                out[s, i, x], size[s, i, x] = p @ vv, p @ vv.abs()
                total[s, i, x] = vv.abs().sum(0)
    return out, size, total


def _check_attention(got, want, what):
    out, size, total = want
    f = torch.finfo(got.dtype)
    err = (got.double().cpu() - out).abs()
    tol = f.eps / 2 * out.abs() + (f.eps + 2.0 ** -12) * size + f.smallest_normal * f.eps / 2
    if got.dtype is torch.float16:
        tol += 2.0 ** -25 * total
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, worst {float(err[bad].max()):.3e}"


def _attention_case(seed, lens, n, heads, kv, dim, dtype, layout, cap=None, trees=None, fill=NAN):
    """Inputs whose unused cache slots hold ``fill``."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    b = len(lens)
    cap = cap or max(lens) + n
    q = (torch.randn(b, n, heads, dim, generator=g) * 1.5).to(dtype)
    k, v = (torch.full((b, kv, cap, dim), fill, dtype=dtype) for _ in range(2))
    trees = trees or [_tree(rng, n) for _ in range(b)]
    for s, length in enumerate(lens):
        if 0 <= length <= cap - n:
            for c in (k, v):
                c[s, :, :length + n] = torch.randn(kv, length + n, dim, generator=g).to(dtype)
    masks = _i64([[_signed(m) for m in _bits(t)] for t in trees])
    return q, k, v, _i64(lens), masks


def _to_cache(t, layout):
    """t on the device in the layout, unused memory around it NaN."""
    b, kv, cap, dim = t.shape
    c = _cache(b, kv, cap, dim, t.dtype, layout, NAN)
    c.copy_(t)
    return c


def _attend(q, k, v, lengths, masks, layout="row", scale=None):
    return _td().tree_attention(q.to(DEV), _to_cache(k, layout),
                                _to_cache(v, "gap" if layout == "gap" else "row"),
                                lengths.to(DEV), masks.to(DEV), scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["row", "col", "gap"])
@pytest.mark.parametrize("n,heads,kv,dim", [
    (1, 4, 4, 64), (1, 8, 1, 128), (4, 12, 4, 128), (16, 4, 1, 128), (25, 4, 2, 256), (64, 2, 1, 64),
    (64, 8, 1, 128), (7, 7, 1, 128), (33, 3, 3, 256), (64, 4, 1, 256), (3, 20, 1, 64), (17, 16, 1, 64)])
def test_attention(dtype, layout, n, heads, kv, dim):
    say(f"attention {dtype} {layout} n={n} heads={heads}/{kv} dim={dim}")
    lens = [0, 1, 130, 63, 64, 65, 300]
    q, k, v, lengths, masks = _attention_case(n * dim, lens, n, heads, kv, dim, dtype, layout,
                                              cap=max(lens) + n + 5)
    got = _attend(q, k, v, lengths, masks, layout)
    _check_attention(got, _attend_ref(q, k, v, lengths, masks, dim ** -0.5), "attention")


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("lens,n,heads,kv,dim", [
    ([5000], 2, 8, 2, 128), ([9001], 9, 4, 1, 128), ([4000, 17], 40, 2, 1, 64),
    ([3000, 0, 2500], 5, 4, 2, 256), ([2047], 64, 8, 1, 128)])
def test_attention_long(lens, n, heads, kv, dim, layout):
    say(f"attention long {lens} n={n} {heads}/{kv} dim={dim} {layout}")
    q, k, v, lengths, masks = _attention_case(11, lens, n, heads, kv, dim, torch.bfloat16, layout)
    got = _attend(q, k, v, lengths, masks, layout)
    _check_attention(got, _attend_ref(q, k, v, lengths, masks, dim ** -0.5), "attention")


def test_attention_empty_slots_and_rows():
    """Empty slots of the batch, sequences too long for the cache, and nodes whose
    mask leaves nothing are zeros; lengths are read on the device."""
    say("attention empty slots")
    lens = [40, -1, 0, 41, 1 << 40, -(1 << 40)]
    n = 9
    q, k, v, lengths, masks = _attention_case(5, [40, 0, 0, 0, 0, 0], n, 4, 2, 128, torch.bfloat16,
                                              "row", cap=49)
    lengths = _i64(lens)
    masks[2, 3] = 0
    masks[0, 4] = 0                        # sees the sequence alone
    masks[0, 5] = _signed((1 << 64) - 1)   # bits from n on are not looked at
    for layout in ("row", "col"):
        got = _attend(q, k, v, lengths, masks, layout)
        _check_attention(got, _attend_ref(q, k, v, lengths, masks, 128 ** -0.5), layout)
        assert float(got[[1, 3, 4, 5]].abs().max()) == 0 and float(got[2, 3].abs().max()) == 0


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("length,n,heads", [(70, 12, 4), (61, 64, 2), (0, 5, 8)])
def test_attention_masked_places(layout, bad, length, n, heads):
    """A drafted token that some nodes see and others do not may hold NaN or
    infinities: the others' results are those of finite inputs."""
    say(f"attention masked {bad} length={length} n={n} {layout}")
    tree = [-1, 0, 0] + [1 + i % 2 for i in range(n - 3)]  # two branches, 1 and 2
    q, k, v, lengths, masks = _attention_case(7, [length], n, heads, 1, 128, torch.bfloat16, layout,
                                              trees=[tree])
    want = _attend_ref(q, k, v, lengths, masks, 128 ** -0.5)
    rows = [i for i in range(n) if not int(masks[0, i]) >> 1 & 1]  # do not see node 1
    for which in ("v", "k", "both"):
        k2, v2 = k.clone(), v.clone()
        if which != "v":
            k2[0, 0, length + 1, ::3] = bad
        if which != "k":
            v2[0, 0, length + 1, ::2] = bad
        got = _attend(q, k2, v2, lengths, masks, layout)
        _check_attention(got[:, rows], [t[:, rows] for t in want], which)
        if which == "v":  # and node 1 itself has it
            seen = got[0, 1, :, ::2].float()
            assert bool((torch.isnan(seen) if bad != bad else seen == bad).all())


def test_attention_large_scores():
    """Scores far apart and far from zero, and all alike."""
    say("attention large scores")
    n, dim = 6, 64
    q, k, v, lengths, masks = _attention_case(9, [200], n, 2, 1, dim, torch.float16, "row")
    for factor in (0.0, 30.0):
        got = _attend(q * factor, k, v, lengths, masks, "row")
        ref = _attend_ref(q * factor, k, v, lengths, masks, dim ** -0.5)
        if factor:  # products of size 64 * 4.5 * 30: fp32 sums are off by 2^-24 * 64 * 200
            ref = (ref[0], ref[1] * 4, ref[2])
        _check_attention(got, ref, f"factor {factor}")
    got = _attend(q, k, v, lengths, masks, "row", scale=0.0)
    _check_attention(got, _attend_ref(q, k, v, lengths, masks, 0.0), "scale 0")


def test_attention_strided_queries_and_shared_inputs():
    """Queries inside a wider tensor, one mask row for all, a cache that all
    sequences share."""
    say("attention strides")
    n, heads, dim = 5, 4, 64
    q, k, v, lengths, masks = _attention_case(13, [50, 50, 50], n, heads, 2, dim, torch.bfloat16,
                                              "row", trees=[[-1, 0, 0, 1, 2]] * 3)
    wide = torch.full((3, n, heads * dim + 64), NAN, dtype=q.dtype, device=DEV)
    wide[:, :, 16:16 + heads * dim] = q.flatten(2).to(DEV)
    qs = wide[:, :, 16:16 + heads * dim].unflatten(2, (heads, dim))
    kd, vd = k[:1].to(DEV).expand(3, -1, -1, -1), v[:1].to(DEV).expand(3, -1, -1, -1)
    got = _td().tree_attention(qs, kd, vd, lengths.to(DEV), masks[0].to(DEV))
    want = _attend_ref(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), lengths, masks,
                       dim ** -0.5)
    _check_attention(got, want, "strides")
    turned = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)  # heads before nodes
    assert torch.equal(_td().tree_attention(turned, kd, vd, lengths.to(DEV), masks.to(DEV)), got)


def test_attention_offsets_past_32_bits():
    """A cache whose last head starts past 4 GiB, and whose positions are far apart."""
    say("attention 64-bit offsets")
    n, dim, cap = 3, 64, 70
    stride = 1 << 25  # elements from one position to the next: 70 of them span 4.7 GB
    store = torch.empty(stride * (cap - 1) + dim, dtype=torch.bfloat16, device=DEV)
    q, k, v, lengths, masks = _attention_case(17, [cap - n], n, 2, 1, dim, torch.bfloat16, "row")
    kd = store.as_strided((1, 1, cap, dim), (8, 8, stride, 1))
    kd.copy_(k)
    got = _td().tree_attention(q.to(DEV), kd, v.to(DEV), lengths.to(DEV), masks.to(DEV))
    want = _attend_ref(q, k, v, lengths, masks, dim ** -0.5)
    _check_attention(got, want, "keys")
    kd.copy_(v)
    got = _td().tree_attention(q.to(DEV), k.to(DEV), kd, lengths.to(DEV), masks.to(DEV))
    _check_attention(got, want, "values")
    col = store.as_strided((1, 1, cap, dim), (8, 8, 1, stride))
    col.copy_(k)
    got = _td().tree_attention(q.to(DEV), col, v.to(DEV), lengths.to(DEV), masks.to(DEV))
    _check_attention(got, want, "keys by dimension")


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def _verify_ref(logits, tokens, u, parents, probs, temps):
    """The walk from node to node in float64."""
    b, n, vocab = logits.shape
    out, path = np.full((b, n), -1), np.full((b, n), -1)
    count = np.zeros(b, np.int64)
    for s in range(b):
        if not 0 <= tokens[s, 0] < vocab:
            continue
        par = [i - 1 for i in range(n)] if parents is None else parents[s].tolist()
        there = [True]
        for i in range(1, n):
            there.append(0 <= tokens[s, i] < vocab and 0 <= par[i] < i and there[par[i]])
        node, steps, said = 0, [0], []
        while True:
            x = logits[s, node].double().numpy()
            x = np.where(np.isnan(x), -INF, x)
            top = x.max()
            if top == -INF:
                left = np.zeros(vocab)
            elif temps[s] > 0:
                with np.errstate(invalid="ignore"):
                    left = np.where(x == top, 1.0, np.exp((x - top) / float(temps[s])))
                left /= left.sum()
            else:
                left = (np.arange(vocab) == x.argmax()).astype(float)
            whole, went = left, None
            for c in [i for i in range(1, n) if there[i] and par[i] == node]:
                t, r = int(tokens[s, c]), float(u[s, c])
                if probs is not None:
                    q = probs[s, node].double().numpy()
                    q = np.where((q > 0) & (q < INF), q, 0.0)
                    ok, rest = r * q[t] < left[t], np.maximum(left - q, 0)
                else:
                    ok, rest = r * (left.sum() if left.sum() else 1) < left[t], left.copy()
                    rest[t] = 0
                if ok:
                    went = c
                    break
                left = rest
            if went is None:
                break
            node = went
            steps.append(went)
            said.append(int(tokens[s, went]))
        if not left.sum() > 0:
            left = whole
        cum = np.cumsum(left)
        hit = np.flatnonzero(cum > float(u[s, 0]) * cum[-1])
        said.append(int(hit[0]) if len(hit) else -1)
        count[s] = len(steps)
        path[s, :len(steps)], out[s, :len(steps)] = steps, said
    return out, path, count


def _verify_case(seed, b, n, vocab, mode, dtype=torch.float32, temps=(0.0, 0.7, 1.0, 1.4), sharp=2.0):
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    logits = (torch.randn(b, n, vocab, generator=g) * sharp).to(dtype)
    temp = torch.tensor([temps[s % len(temps)] for s in range(b)])
    u = torch.rand(b, n, generator=g)
    tokens = torch.randint(0, vocab, (b, n), generator=g)
    parents = probs = None
    if mode == "tree":
        parents = _i64([_tree(rng, n) for _ in range(b)])
        for s in range(b):  # a node's likeliest tokens, one after the other
            for i in range(1, n):
                p = int(parents[s, i])
                rank = parents[s, 1:i].tolist().count(p)
                order = logits[s, p].float().argsort(descending=True, stable=True)
                tokens[s, i] = order[min(rank, vocab - 1)]
    elif mode == "probs" and n > 1:
        probs = torch.softmax(logits[:, :-1].float() + 0.5 * torch.randn(b, n - 1, vocab, generator=g), -1)
        tokens[:, 1:] = torch.multinomial(probs.reshape(-1, vocab), 1, generator=g).view(b, n - 1)
    return logits, tokens, u, parents, probs, temp


def _check_verify(logits, tokens, u, parents, probs, temp, what=""):
    dev = [t if t is None else t.to(DEV) for t in (logits, tokens, u, parents, probs, temp)]
    got = _td().verify_drafts(dev[0], dev[1], dev[2], parents=dev[3], draft_probs=dev[4],
                              temperature=dev[5])
    want = _verify_ref(logits, tokens, u, parents, probs, temp)
    for x, y, name in zip(got, want, ("out", "path", "count")):
        assert x.tolist() == y.tolist(), f"{what} {name}"
    return got


@pytest.mark.parametrize("mode", ["tree", "chain", "probs"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,n,vocab", [
    (5, 1, 1), (4, 3, 2), (8, 5, 63), (9, 17, 1000), (4, 64, 300), (6, 33, 4097), (4, 8, 8192),
    (5, 4, 8193), (4, 5, 20001), (40, 6, 12288)])
def test_verify(mode, dtype, b, n, vocab):
    say(f"verify {mode} {dtype} b={b} n={n} vocab={vocab}")
    _check_verify(*_verify_case(b * n + vocab, b, n, vocab, mode, dtype))


def test_verify_large_vocabulary():
    say("verify large vocabulary")
    for mode in ("tree", "probs"):
        _check_verify(*_verify_case(3, 3, 4, 151936, mode, temps=(1.0, 0.8)), what=mode)
    _check_verify(*_verify_case(4, 1, 1, 1 << 20, "chain", temps=(1.0,)), what="one token")


@pytest.mark.parametrize("mode", ["tree", "chain", "probs"])
def test_verify_padded(mode):
    """Absent nodes and empty slots; filtered, NaN and infinite logits; equal largest
    logits; numbers at the ends of their range."""
    say(f"verify padded {mode}")
    b, n, vocab = 14, 7, 500
    logits, tokens, u, parents, probs, temp = _verify_case(21, b, n, vocab, mode, sharp=1.0)
    tokens[0, 3:] = -1
    tokens[1] = -1
    tokens[2, 1] = vocab
    tokens[3, 0] = vocab + 5
    if parents is not None:
        parents[4, 2:] = -1
        parents[5, 3], parents[5, 4] = 3, 6
    keep = torch.rand(vocab, generator=torch.Generator().manual_seed(1)) < 0.02
    logits[6:9] = torch.where(keep, logits[6:9], -INF)
    logits[9, :, ::7] = NAN
    logits[10, :2] = -INF
    logits[11, :, 5] = INF
    logits[11, :, 250] = INF
    logits[12] = 0.0
    u[6], u[12], u[7, 0] = 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24
    if probs is not None:
        probs[8, :, ::3], probs[9, :, ::5] = NAN, -1.0
        probs[12] = torch.softmax(logits[12, :-1], -1)
    _check_verify(logits, tokens, u, parents, probs, temp, mode)


def test_verify_repeated_and_exhausted_siblings():
    """A token drafted twice is rejected twice; siblings that hold all of the
    distribution are accepted one way or another."""
    say("verify siblings")
    n, vocab = 6, 4
    b = 64
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(b, n, vocab, generator=g)
    logits[:, 0, 3] = -INF
    tokens = _i64([[0, 0, 0, 1, 1, 2]]).expand(b, n).contiguous()
    parents = _i64([-1, 0, 0, 0, 0, 0]).expand(b, n).contiguous()
    u = torch.rand(b, n, generator=g)
    got = _check_verify(logits, tokens, u, parents, None, torch.ones(b))
    assert set(got[2].tolist()) == {2}  # tokens 0, 1, 2 are all there is


def test_verify_layouts():
    """Strided and unaligned logits and probabilities, one tree for all, a number as
    temperature, repeated calls."""
    say("verify layouts")
    b, n, vocab = 3, 5, 777
    logits, tokens, u, parents, probs, temp = _verify_case(31, b, n, vocab, "probs", temps=(1.0,))
    td = _td()
    want = _verify_ref(logits, tokens, u, None, probs, temp)
    wide = torch.full((n, b, vocab + 9), NAN, device=DEV)
    wide[:, :, 3:3 + vocab] = logits.transpose(0, 1).to(DEV)
    lt = wide.transpose(0, 1)[:, :, 3:3 + vocab]
    pw = torch.full((b, n, vocab + 2), NAN, device=DEV)
    pw[:, 1:, 1:-1] = probs.to(DEV)
    for lg in (lt, lt.transpose(1, 2).contiguous().transpose(1, 2)):
        for _ in range(2):
            got = td.verify_drafts(lg, tokens.to(DEV), u.to(DEV), draft_probs=pw[:, 1:, 1:-1])
            for x, y in zip(got, want):
                assert x.tolist() == y.tolist()
    logits, tokens, u, parents, _, temp = _verify_case(32, b, n, vocab, "tree", temps=(0.5,))
    parents[:] = parents[0]
    got = td.verify_drafts(logits.to(DEV), tokens.to(DEV), u.to(DEV), parents=parents[0].to(DEV),
                           temperature=0.5)
    for x, y in zip(got, _verify_ref(logits, tokens, u, parents, None, temp)):
        assert x.tolist() == y.tolist()


@pytest.mark.parametrize("mode", ["tree", "probs"])
def test_verify_keeps_the_distribution(mode):
    """The first token that a step adds has the target's distribution, whatever the
    drafts: 40,000 sequences, each frequency within 5 standard deviations."""
    say(f"verify distribution {mode}")
    b, vocab, g = 40000, 6, torch.Generator(device=DEV).manual_seed(77)
    row = torch.tensor([0.3, -1.0, 1.2, 0.0, -0.4, 0.9], device=DEV)
    n = 4 if mode == "tree" else 2
    logits = row.expand(b, n, vocab)
    u = torch.rand(b, n, generator=g, device=DEV)
    if mode == "tree":  # three drafts for the one place
        tokens = _i64([0, 2, 0, 4]).to(DEV).expand(b, n).contiguous()
        out, _, _ = _td().verify_drafts(logits, tokens, u, parents=_i64([-1, 0, 0, 0]).to(DEV))
    else:
        q = torch.softmax(-row, 0)
        tokens = torch.multinomial(q.expand(b, vocab), 2, replacement=True, generator=g)
        out, _, _ = _td().verify_drafts(logits, tokens, u, draft_probs=q.expand(b, 1, vocab))
    p = torch.softmax(row.double(), 0).cpu()
    freq = torch.bincount(out[:, 0].cpu(), minlength=vocab).double() / b
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / b).sqrt()).all()), (freq, p)


# ---------------------------------------------------------------------------
# accepted rows to the front
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["row", "col", "gap"])
@pytest.mark.parametrize("n,dim,layers", [(1, 128, None), (9, 64, 3), (64, 128, 2), (33, 256, None)])
def test_keep_accepted(dtype, layout, n, dim, layers):
    say(f"keep {dtype} {layout} n={n} dim={dim} layers={layers}")
    rng, g = random.Random(n), torch.Generator().manual_seed(n)
    lens, kv = [0, 5, 9, -1, 10, 3, 4], 3
    b, cap = len(lens), n + 9
    path, count = torch.full((b, n), -1), torch.zeros(b, dtype=torch.int64)
    for s in range(b):
        p = [0] + sorted(rng.sample(range(1, n), rng.randint(0, n - 1)))
        path[s, :len(p)], count[s] = _i64(p), len(p)
    count[5] = 0
    vlay = "gap" if layout == "gap" else "row"
    k, v = (_cache(b, kv, cap, dim, dtype, y, 0.0, g, layers) for y in (layout, vlay))
    want = []
    for c in (k, v):
        w = c.cpu().clone()
        w5 = w if layers else w[None]
        for s, length in enumerate(lens):
            if 0 <= length <= cap - n:
                src = [length + int(p) for p in path[s, :int(count[s])]]
                w5[:, s, :, length:length + len(src)] = w5[:, s][:, :, src].clone()
        want.append(w)
    _td().keep_accepted(k, v, _i64(lens).to(DEV), path.to(DEV), count.to(DEV))
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_keep_follows_only_ascending_paths():
    say("keep: paths that are none")
    n, cap = 8, 20
    k = torch.arange(cap, dtype=torch.float32).to(torch.bfloat16)[None, None, :, None].expand(5, 1, cap, 64)
    k, v = k.contiguous().to(DEV), k.contiguous().to(DEV)
    path = _i64([[0, 2, 1, 3, 4, 5, 6, 7], [0, 3, 9, 9, 9, 9, 9, 9], [0, 2, -5, 4, 5, 6, 7, 7],
                 [1, 3, 3, 4, 5, 6, 7, 7], [0, 1, 2, 3, 4, 5, 6, 7]])
    count = _i64([8, 3, 8, 3, 1 << 40])
    _td().keep_accepted(k, v, _i64([4] * 5).to(DEV), path.to(DEV), count.to(DEV))
    got = k[:, 0, :, 0].float().cpu() - torch.arange(cap)
    want = torch.zeros(5, cap)
    want[0, 5], want[1, 5], want[2, 5], want[3, 4], want[3, 5] = 1, 2, 1, 1, 2
    assert torch.equal(got, want) and torch.equal(k, v)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def _round(td, s):
    plan = td.tree_plan(s["parents"], s["lengths"])
    b, n = s["tokens"].shape
    outs = []
    for i, qkv in enumerate(s["qkv"]):
        q = td.qk_norm_rope_write(qkv, s["heads"], s["kv"], s["table"], plan.positions, s["k"][i],
                                  s["v"][i], s["lengths"], s["w"], s["w"], EPS)
        outs.append(td.tree_attention(q.view(b, n, s["heads"], -1), s["k"][i], s["v"][i],
                                      s["lengths"], plan.masks))
    out, path, count = td.verify_drafts(s["logits"], s["tokens"], s["u"], parents=s["parents"])
    td.keep_accepted(s["k"], s["v"], s["lengths"], path, count)
    s["lengths"].add_(count)
    return torch.stack(outs), out, path, count


def _round_state(seed, lens, n, layout, dtype=torch.bfloat16, layers=2, vocab=900):
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    b, heads, kv, dim, cap = len(lens), 4, 2, 128, max(lens) + 3 * n
    logits, tokens, u, _, _, _ = _verify_case(seed, b, n, vocab, "tree")
    return {"heads": heads, "kv": kv, "parents": _i64([_tree(rng, n) for _ in lens]).to(DEV),
            "lengths": _i64(lens).to(DEV), "logits": logits.to(DEV), "tokens": tokens.to(DEV),
            "u": u.to(DEV), "table": torch.rand(cap, dim, generator=g).to(DEV),
            "w": (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).to(DEV),
            "qkv": [torch.randn(b * n, (heads + 2 * kv) * dim, generator=g).to(dtype).to(DEV)
                    for _ in range(layers)],
            "k": _cache(b, kv, cap, dim, dtype, layout, 0.0, g, layers),
            "v": _cache(b, kv, cap, dim, dtype, "row", 0.0, g, layers)}


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("layout", ["row", "col"])
def test_round_against_reference(layout):
    """A step as it is used: every stage against the float64 statements, fed with
    what the stage before it left."""
    say(f"round {layout}")
    td, n, lens = _td(), 11, [30, 0, 64]
    s = _round_state(3, lens, n, layout)
    before = [s["k"].clone(), s["v"].clone()]
    q_in = [t.cpu() for t in s["qkv"]]
    outs, out, path, count = _round(td, s)
    masks = [_bits(t) for t in s["parents"].tolist()]
    pos = _i64([[length + bin(m).count("1") - 1 for m in ms] for length, ms in zip(lens, masks)])
    signed = _i64([[_signed(m) for m in ms] for ms in masks])
    w = s["w"].cpu()
    want_v = _verify_ref(s["logits"].cpu(), s["tokens"].cpu(), s["u"].cpu(), s["parents"].cpu(), None,
                         torch.ones(3))
    for x, y in zip((out, path, count), want_v):
        assert x.tolist() == y.tolist()
    assert s["lengths"].tolist() == [a + int(c) for a, c in zip(lens, count)]
    for i, qkv in enumerate(q_in):
        (q, _), (k, _) = _rope_ref(qkv, 4, 2, s["table"].cpu(), pos.view(-1), w, w)
        kc, vc = (c[i].cpu().clone() for c in before)
        rows = qkv.view(3, n, 8, 128)
        for b, length in enumerate(lens):
            kc[b, :, length:length + n] = k.view(3, n, 2, 128)[b].transpose(0, 1).to(kc.dtype)
            vc[b, :, length:length + n] = rows[b, :, 6:].transpose(0, 1)
        ref = _attend_ref(q.view(3, n, 4, 128).to(kc.dtype), kc, vc, _i64(lens), signed, 128 ** -0.5)
        # queries and keys may each sit on the other side of a rounding: a score of up
        # to 40 is off by 2^-8 of it at most where all its products are, 2^-3 in all
        _check_attention(outs[i], (ref[0], ref[1] * (1 + 2.0 ** 5), ref[2]), f"layer {i}")
        for b, length in enumerate(lens):
            src = [length + p for p in path[b].tolist() if p >= 0]
            vc[b, :, length:length + len(src)] = vc[b][:, src]
        assert torch.equal(s["v"][i].cpu(), vc)


def test_round_in_a_graph():
    """A captured step replayed with the program's own work between the replays: the
    lengths move on, every replay as the eager step from the same state."""
    say("round in a graph")
    td, n, lens = _td(), 6, [12, 3]
    a, b = _round_state(9, lens, n, "col"), _round_state(9, lens, n, "col")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _round(td, _round_state(9, lens, n, "col"))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = _round(td, a)
    torch.cuda.synchronize()
    for r in range(4):
        fresh = torch.rand(2, n, generator=torch.Generator().manual_seed(r)).to(DEV)
        for s in (a, b):
            s["u"].copy_(fresh)
            s["lengths"].copy_(_i64([12 + r, 3]).to(DEV))
        graph.replay()
        want = _round(td, b)
        torch.cuda.synchronize()
        assert _same(got, want), f"replay {r}"
        for name in ("k", "v", "lengths"):
            assert torch.equal(a[name], b[name]), f"replay {r}: {name}"


def test_round_on_two_streams():
    """Steps of two batches on two streams at once, each as alone."""
    say("round on two streams")
    td, n = _td(), 16
    args = [(5, [900, 20]), (6, [40, 1500])]
    want = [_round(td, _round_state(seed, lens, n, "row")) for seed, lens in args]
    states = [[_round_state(seed, lens, n, "row") for _ in range(4)] for seed, lens in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for r in range(4):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(_round(td, states[k][r]))
    torch.cuda.synchronize()
    for k in range(2):
        for one in got[k]:
            assert _same(one, want[k])


def test_inference_tensors_and_versions():
    say("inference tensors")
    td = _td()
    with torch.inference_mode():
        s = _round_state(2, [4, 5], 3, "row")
        _round(td, s)
    s = _round_state(2, [4, 5], 3, "row")
    v = s["k"]._version
    _round(td, s)
    assert s["k"]._version > v


def test_refusals():
    say("refusals")
    td = _td()
    n, heads, kv, dim, cap = 3, 4, 2, 64, 16
    k = torch.zeros(2, kv, cap, dim, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, n, heads, dim, dtype=torch.bfloat16, device=DEV)
    lengths, masks = _i64([1, 1]).to(DEV), torch.ones(2, n, dtype=torch.int64, device=DEV)
    qkv = torch.zeros(2 * n, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device=DEV)
    table, pos = torch.zeros(cap, dim, device=DEV), torch.zeros(2 * n, dtype=torch.int64, device=DEV)
    attend = [
        (TypeError, (q.float(), k, k, lengths, masks)),
        (TypeError, (q.half(), k, k, lengths, masks)),
        (TypeError, (q, k, k, lengths.int(), masks)),
        (TypeError, (q, k, k, lengths, masks.int())),
        (ValueError, (q, k, k[:1], lengths, masks)),
        (ValueError, (q[:1], k, k, lengths, masks)),
        (ValueError, (q[..., :32], k, k, lengths, masks)),
        (ValueError, (q[:, :, :3], k, k, lengths, masks)),
        (ValueError, (q, k, k, lengths[:1], masks)),
        (ValueError, (q, k, k, lengths, masks[:, :2])),
        (ValueError, (q, k, k.transpose(-1, -2).contiguous().transpose(-1, -2), lengths, masks)),
        (ValueError, (q[:, :0], k, k, lengths, masks[:, :0])),
        (ValueError, (q[:, :1].expand(2, 65, heads, dim), k, k, lengths, masks)),
        (RuntimeError, (q, k, k[..., :1].expand(2, kv, cap, dim + 1)[..., 1:], lengths, masks)),
        (RuntimeError, (q.cpu(), k, k, lengths, masks)),
        (RuntimeError, (q.clone().requires_grad_(), k, k, lengths, masks)),
    ]
    for err, args in attend:
        with pytest.raises((err, ValueError)):
            td.tree_attention(*args)
    odd = torch.zeros(2, n, heads, 80, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="dimensions"):
        td.tree_attention(odd, *[torch.zeros(2, kv, cap, 80, dtype=torch.bfloat16, device=DEV)] * 2,
                          lengths, masks)
    shifted = torch.zeros(2, kv, cap, dim + 4, dtype=torch.bfloat16, device=DEV)[..., 4:]
    with pytest.raises(RuntimeError, match="aligned"):
        td.tree_attention(q, shifted, k, lengths, masks)
    rope = [
        (TypeError, (qkv.float(), heads, kv, table, pos)),
        (TypeError, (qkv, heads, kv, table.half(), pos)),
        (TypeError, (qkv, heads, kv, table, pos.int())),
        (ValueError, (qkv, heads, kv + 1, table, pos)),
        (ValueError, (qkv, heads, kv, table, pos[:-1])),
        (ValueError, (qkv, heads, kv, table, pos, torch.ones(dim, device=DEV))),
        (RuntimeError, (qkv, heads, kv, table[:, :24], pos)),
        (RuntimeError, (qkv, heads, kv, torch.zeros(cap, 2 * dim, device=DEV), pos)),
    ]
    for err, args in rope:
        with pytest.raises(err):
            td.qk_norm_rope(*args)
    for bad in (k[:1].expand(2, -1, -1, -1), k[:, :1].expand(-1, kv, -1, -1),
                k.flatten()[:2 * kv * cap * dim // 2].as_strided(k.shape, (kv * cap * dim // 2, cap * dim // 2, 8, 1))):
        with pytest.raises(ValueError, match="overlaps"):
            td.qk_norm_rope_write(qkv, heads, kv, table, pos, bad, k, lengths)
        with pytest.raises(ValueError, match="overlaps"):
            td.keep_accepted(k, bad, lengths, masks, lengths)
    with pytest.raises(ValueError):
        td.qk_norm_rope_write(qkv[:5], heads, kv, table, pos[:5], k, k.clone(), lengths)
    logits = torch.zeros(2, n, 50, device=DEV)
    tok, u = torch.zeros(2, n, dtype=torch.int64, device=DEV), torch.zeros(2, n, device=DEV)
    probs = torch.zeros(2, n - 1, 50, device=DEV)
    for err, args, kw in [
            (TypeError, (logits.double(), tok, u), {}), (TypeError, (logits, tok.int(), u), {}),
            (ValueError, (logits, tok[:, :2], u), {}), (ValueError, (logits, tok, u.double()), {}),
            (ValueError, (logits[0], tok, u), {}), (ValueError, (logits, tok, u), {"temperature": -1.0}),
            (ValueError, (logits, tok, u), {"temperature": NAN}),
            (ValueError, (logits, tok, u), {"temperature": u}),
            (ValueError, (logits, tok, u), {"parents": tok, "draft_probs": probs}),
            (ValueError, (logits, tok, u), {"draft_probs": probs[:, :1]}),
            (ValueError, (logits, tok, u), {"draft_probs": probs.half()}),
            (TypeError, (logits, tok, u), {"parents": tok.int()})]:
        with pytest.raises(err):
            td.verify_drafts(*args, **kw)
    with pytest.raises(ValueError):
        td.tree_plan(tok[:, :0], lengths)
    with pytest.raises(TypeError):
        td.tree_plan(tok.int(), lengths)
    # nothing to do
    assert td.tree_attention(q[:0], k[:0], k[:0], lengths[:0], masks[:0]).shape == (0, n, heads, dim)
    assert [t.shape[0] for t in td.verify_drafts(logits[:0], tok[:0], u[:0])] == [0, 0, 0]
    assert td.tree_plan(tok[:0], lengths[:0]).masks.shape == (0, n)


@pytest.mark.parametrize("heads,kv,dim,layout", [(4, 4, 128, "col"), (8, 2, 256, "row"), (16, 1, 64, "row")])
def test_attention_many_sequences(heads, kv, dim, layout):
    """More sequences than a wave has lanes, empty slots among them, several to a
    workgroup."""
    say(f"attention many sequences {heads}/{kv} dim={dim} {layout}")
    rng, n = random.Random(dim), 3
    lens = [rng.choice([-1, 0, 1, 5, 61, 62, 100, 200]) for _ in range(200)]
    q, k, v, lengths, masks = _attention_case(dim, lens, n, heads, kv, dim, torch.bfloat16, layout,
                                              cap=203)
    got = _attend(q, k, v, lengths, masks, layout)
    _check_attention(got, _attend_ref(q, k, v, lengths, masks, dim ** -0.5), "attention")


def test_strides_along_one_element_are_not_looked_at():
    say("strides along one element")
    q, k, v, lengths, masks = _attention_case(3, [20], 2, 2, 1, 64, torch.bfloat16, "row")
    want = _attend(q, k, v, lengths, masks)
    kd, vd = (t.to(DEV).as_strided(t.shape, (3, 5, 64, 1)) for t in (k, v))
    qd = q.to(DEV).as_strided(q.shape, (7, 128, 64, 1))
    assert torch.equal(_td().tree_attention(qd, kd, vd, lengths.to(DEV), masks.to(DEV)), want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("n,group", [(5, 13), (32, 4), (28, 7), (25, 8), (64, 7)])
def test_attention_row_blocks(n, group, dim, layout):
    """Rows of a KV head around and past a workgroup's: 65, 128, 196, 200, 448."""
    say(f"attention rows {n * group} dim={dim} {layout}")
    q, k, v, lengths, masks = _attention_case(n + dim, [190, 0, 700], n, group, 1, dim, torch.bfloat16,
                                              layout)
    got = _attend(q, k, v, lengths, masks, layout)
    _check_attention(got, _attend_ref(q, k, v, lengths, masks, dim ** -0.5), "attention")


def test_attention_more_row_blocks_than_workgroups():
    """4096 query heads of one KV head: every row block goes through the whole line."""
    say("attention row blocks")
    n, dim = 17, 64
    q, k, v, lengths, masks = _attention_case(2, [100, -1, 70, 0], n, 4, 1, dim, torch.bfloat16, "row",
                                              cap=120)
    want = _attend_ref(q, k, v, lengths, masks, dim ** -0.5)
    got = _attend(q.repeat(1, 1, 1024, 1), k, v, lengths, masks)
    for h in (0, 1, 7, 2046, 4095):
        _check_attention(got[:, :, h:h + 1], [t[:, :, h % 4:h % 4 + 1] for t in want], f"head {h}")
    assert torch.equal(got[:, :, :4].repeat(1, 1, 1024, 1), got)
