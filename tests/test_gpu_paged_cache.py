"""GPU tests of the paged 8-bit cache (polarengine_vllm.kernels.paged_cache) against
float64 and whole-number statements of the same inputs on the CPU.

Tolerances. Plans, slots, scales and codes are whole numbers or exact roundings and
have to be equal. Attention: a result rounded once to 16 bits is off by at most half a
step, h = finfo.eps / 2 of its value (and half the smallest subnormal). Each
probability may be rounded to fp16 (2^-11 of itself), in the sum of the values and,
alike or not, in the sum that divides them: at most 2 * 2^-11 of A = sum p |v| / sum p
together. fp32 scores are sums of at most 256 products; codes are at most 448 times a
power of two, so with |score| <= 40 and sums of magnitudes up to 8 times that their
error is below 256 * 2^-24 * 320 * 2^-7 < 2^-11 in the exponent even if no rounding
cancels: 2^-11 A more. A probability that fp16 cannot hold adds 2^-25 of the largest."""

import math
import random

import numpy as np
import pytest
import torch

from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu

NAN = float("nan")
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LEAST = -100


def _pc():
    from polarengine_vllm.kernels import paged_cache
    return paged_cache


def _i64(x):
    return torch.tensor(x, dtype=torch.int64)


# ---------------------------------------------------------------------------
# plan and release
# ---------------------------------------------------------------------------
def _plan_ref(lengths, counts, tables, free, count, rows, t):
    starts, pos, slots, after = [0], [-1] * rows, [-1] * rows, []
    wanted = taken = 0
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    top = max(0, min(count, len(free)))
    for b, (n, c) in enumerate(zip(lengths, counts)):
        c = max(c, 0) if n >= 0 else 0
        first = starts[-1]
        starts.append(first + c)
        ok = n >= 0 and n + c <= width * t and first + c <= rows
        lacks = [j for j in range(n // t, (n + c - 1) // t + 1) if tables[b][j] < 0] if ok and c else []
        wanted += len(lacks)
        ok = ok and (not lacks or wanted <= top)
        after.append(n + c if ok else -1)
        if ok:
            for j in lacks:
                tables[b][j] = free[top - 1 - taken]
                taken += 1
            for i in range(c):
                pos[first + i] = n + i
                slots[first + i] = tables[b][(n + i) // t] * t + (n + i) % t
    return [min(s, rows) for s in starts], pos, slots, after, tables, top - taken


def _run_plan(lengths, counts, tables, free, count, rows, t, wide=0):
    """The plan on the GPU and by the reference; both have to agree."""
    pc = _pc()
    d_free, d_count = torch.tensor(free, dtype=torch.int32, device=DEV), _i64([count]).to(DEV)
    d_tables = torch.tensor(tables, dtype=torch.int32).reshape(len(tables), -1)
    d_tables = torch.nn.functional.pad(d_tables, (0, wide), value=77).to(DEV)[:, :d_tables.shape[1]]
    plan = pc.plan_step(_i64(lengths).to(DEV), _i64(counts).to(DEV), d_tables, d_free, d_count, rows, t)
    want = _plan_ref(lengths, counts, tables, free, count, rows, t)
    got = [x.tolist() for x in plan] + [d_tables.tolist(), d_count.item()]
    for name, g, w in zip(("starts", "positions", "slots", "lengths", "tables", "free_count"), got, want):
        assert g == w, f"{name}"
    assert d_free.tolist() == free
    return plan, d_tables, d_free, d_count


def _pool(rng, lengths, t, width, spare):
    """Tables that hold the lengths, and the blocks that are left."""
    have = [-(-max(n, 0) // t) for n in lengths]
    ids = list(range(sum(have) + spare))
    rng.shuffle(ids)
    tables = []
    for n in have:
        tables.append(ids[:n] + [-1] * (width - n))
        ids = ids[n:]
    return tables, ids


@pytest.mark.parametrize("t", [16, 32, 64, 128])
@pytest.mark.parametrize("batch,most,rows", [(1, 1, 1), (3, 5, 16), (64, 1, 64), (70, 40, 900),
                                             (1030, 3, 2500), (4096, 1, 4096), (5, 3000, 9000)])
def test_plan(t, batch, most, rows):
    say(f"plan t={t} batch={batch} most={most} rows={rows}")
    rng = random.Random(batch * t)
    lengths = [rng.choice([-1, 0, t - 1, t, rng.randrange(20 * t)]) for _ in range(batch)]
    counts = [rng.choice([0, 1, most, rng.randrange(most + 1)]) for _ in range(batch)]
    width = 22 + most // t
    tables, free = _pool(rng, lengths, t, width, 8 + batch + batch * (most // t + 1))
    plan, d_tables, d_free, d_count = _run_plan(lengths, counts, tables, free, len(free), rows, t, wide=3)
    # taken back: the pool is as it was
    _pc().release_blocks(d_tables, _i64(lengths).to(DEV), d_free, d_count, t)
    assert d_tables.tolist() == tables and d_free.tolist() == free and d_count.item() == len(free)


@pytest.mark.parametrize("spare", [0, 1, 2, 3, 7])
def test_plan_without_room(spare):
    """Blocks run out, in order; sequences that need none still get their rows."""
    say(f"plan without room, {spare} blocks")
    t = 16
    lengths, counts = [16, 5, 32, -1, 0, 48, 7, 40], [1, 3, 20, 4, 0, 16, 11, 8]
    tables, free = _pool(random.Random(spare), lengths, t, 6, spare)
    _run_plan(lengths, counts, tables, free + [-7] * 3, spare, 80, t)  # an empty stack has room too


def test_plan_refuses_rows_and_positions():
    t = 16
    big = 1 << 40
    for lengths, counts, rows in [([0, 0, 0], [5, 6, 7], 12), ([0, 60, 0], [5, 5, 7], 40),
                                  ([0, big, 0], [5, 5, 7], 40), ([3, 3, 3], [big, 1, 1], 40),
                                  ([3, 3, 3], [1, big, 1], 40), ([3, 3], [-big, 2], 40), ([2, 3], [1, 1], 0),
                                  ([-big, 63, 64], [4, 1, 1], 9), ([64, 64], [0, 1], 5)]:
        say(f"plan {lengths} {counts} rows={rows}")
        tables, free = _pool(random.Random(4), [min(max(n, 0), 64) for n in lengths], t, 4, 30)
        _run_plan(lengths, counts, tables, free, 30, rows, t)


def test_plan_keeps_blocks_that_are_there():
    """Blocks that an earlier plan took (drafts that were turned down) are kept, also
    past the length; missing ones between are filled."""
    tables = [[4, 7, -1, 9, -1, -1], [2, -1, -1, -1, -1, -1]]
    _run_plan([10, 16], [60, 40], tables, [1, 3, 5, 6, 8, 11], 6, 128, 16)


@pytest.mark.parametrize("count", [-5, 0, 4, 99])
def test_plan_count_outside_the_stack(count):
    """A count that the stack cannot hold is taken for what it can."""
    _run_plan([0, 0], [16, 16], [[-1] * 3, [-1] * 3], [5, 6, 7], count, 40, 16)


def test_release():
    pc = _pc()
    t = 32
    rng = random.Random(1)
    for batch in (1, 9, 1500):
        say(f"release batch={batch}")
        lengths = [rng.randrange(-1, 40 * t) for _ in range(batch)]
        tables, ids = _pool(rng, lengths, t, 42, 3)
        keep = [rng.choice([-1, 0, 1, n, n // 2, n + 100, 1 << 40]) for n in lengths]
        cap = len(ids) + sum(len([x for x in r if x >= 0]) for r in tables)
        free = ids + [-7] * (cap - len(ids))
        d_tables = torch.tensor(tables, dtype=torch.int32, device=DEV)
        d_free, d_count = torch.tensor(free, dtype=torch.int32, device=DEV), _i64([len(ids)]).to(DEV)
        pc.release_blocks(d_tables, _i64(keep).to(DEV), d_free, d_count, t)
        back = []
        for b, k in enumerate(keep):
            for j in range(-(-k // t) if k >= 0 else 42, 42):
                if tables[b][j] < 0:
                    break
                back.append(tables[b][j])
                tables[b][j] = -1
        free[len(ids):len(ids) + len(back)] = back[::-1]
        assert d_tables.tolist() == tables
        assert d_free.tolist() == free and d_count.item() == len(ids) + len(back)


def test_release_into_a_full_stack_moves_nothing():
    pc = _pc()
    tables = torch.tensor([[1, 2, -1], [3, -1, -1]], dtype=torch.int32, device=DEV)
    free, count = torch.tensor([0, 4, 9], dtype=torch.int32, device=DEV), _i64([1]).to(DEV)
    pc.release_blocks(tables, _i64([0, 0]).to(DEV), free, count, 16)
    assert tables.tolist() == [[1, 2, -1], [3, -1, -1]] and free.tolist() == [0, 4, 9] and count.item() == 1
    pc.release_blocks(tables, _i64([16, 0]).to(DEV), free, count, 16)
    assert tables.tolist() == [[1, -1, -1], [-1, -1, -1]] and free.tolist() == [0, 3, 2] and count.item() == 3


# ---------------------------------------------------------------------------
# the write
# ---------------------------------------------------------------------------
def _exp(amax):
    e = LEAST
    if amax > 0:
        e = max(LEAST, math.frexp(amax / 448.0)[1] - 1)
        if amax > math.ldexp(448.0, e):
            e += 1
    return e


def _grid(x):
    """Nearest e4m3 values of float64 numbers within 448, ties to even."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    with np.errstate(invalid="ignore"):
        return np.rint(x / step) * step


def _write_ref(codes, exps, x, slots, t, by_dim):
    """codes float64 [blocks, heads, ...], exps int [blocks, heads], x float64 [rows,
    heads, dim]: changed in place."""
    if by_dim:
        codes = codes.swapaxes(-1, -2)
    i, n_slots = 0, codes.shape[0] * t
    while i < len(slots):
        s, n = slots[i], 1
        if not 0 <= s < n_slots:
            i += 1
            continue
        while i + n < len(slots) and slots[i + n] == s + n and (s + n) // t == s // t:
            n += 1
        block, off = s // t, s % t
        for h in range(x.shape[1]):
            rows = x[i:i + n, h]
            fine = np.isfinite(rows)
            e = _exp(float(np.abs(rows[fine]).max())) if fine.any() else LEAST
            if off:
                old = int(exps[block, h])
                e = max(e, old)
                if e > old:
                    codes[block, h] = _grid(np.ldexp(codes[block, h], old - e))
            exps[block, h] = e
            codes[block, h, off:off + n] = np.where(fine, _grid(np.ldexp(rows, -e)), NAN)
        i += n


def _random_cache(g, blocks, kv, t, d, spread=6):
    """Codes of any value (NaN now and then) and scales, on the CPU."""
    pc = _pc()
    k = torch.randint(0, 256, (blocks, kv, t, d), generator=g, dtype=torch.uint8)
    v = torch.randint(0, 256, (blocks, kv, d, t), generator=g, dtype=torch.uint8)
    s = [torch.randint(127 - spread, 127 + spread, (blocks, kv), generator=g).to(torch.uint8) for _ in range(2)]
    return pc.PagedCache(k.view(F8), v.view(F8), s[0].view(E8), s[1].view(E8))


def _check_write(cache, k, v, slots, t, dev_args=None):
    pc = _pc()
    dev = pc.PagedCache(*(x.to(DEV) for x in cache))
    pc.write_blocks(*(dev_args or (k.to(DEV), v.to(DEV))), dev, _i64(slots).to(DEV))
    for codes, scale, x, by_dim, got_c, got_s in [(cache.k, cache.k_scale, k, False, dev.k, dev.k_scale),
                                                 (cache.v, cache.v_scale, v, True, dev.v, dev.v_scale)]:
        want = codes.float().double().numpy()
        exps = scale.view(torch.uint8).numpy().astype(int) - 127
        _write_ref(want, exps, x.double().numpy(), slots, t, by_dim)
        assert np.array_equal(got_s.view(torch.uint8).cpu().numpy().astype(int) - 127, exps)
        np.testing.assert_array_equal(got_c.cpu().float().double().numpy(), want)
    return dev


def _values(g, rows, kv, d, dtype, wild):
    x = torch.randn(rows, kv, d, generator=g)
    x *= 2.0 ** torch.randint(-12, 9, (rows, 1, 1), generator=g)
    if wild:
        u = torch.rand(rows, kv, d, generator=g)
        x = torch.where(u < 0.01, float("inf"), torch.where(u < 0.02, NAN, torch.where(u < 0.03, 0.0, x)))
    return x.to(dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write(d, t, dtype):
    """Runs of every kind: into a block's middle, over block ends, single tokens, rows
    that go nowhere, into blocks with NaN codes, scales that grow and that do not."""
    g = torch.Generator().manual_seed(d + t)
    kv = {64: 5, 128: 2, 256: 1}[d]
    blocks = 14
    cache = _random_cache(g, blocks, kv, t, d)
    order = torch.randperm(blocks, generator=g).tolist()
    slots = []
    for start, n in [(3, 2 * t + 5), (0, t), (t - 1, 1), (0, 1), (5, 1), (t // 2, t // 2 + 1)]:
        slots += [order[p // t] * t + p % t for p in range(start, start + n)] + [-1]
        order = order[(start + n - 1) // t + 1:]
    slots += [blocks * t, blocks * t + 7, -(1 << 40), 1 << 40]
    for wild in (False, True):
        say(f"write d={d} t={t} {dtype} rows={len(slots)} wild={wild}")
        _check_write(cache, _values(g, len(slots), kv, d, dtype, wild), _values(g, len(slots), kv, d, dtype, wild),
                     slots, t)


def test_write_roundings():
    """Every 16-bit value of some binades in a block whose scale is known."""
    t, d = 128, 128
    for dtype in (torch.bfloat16, torch.float16):
        say(f"write roundings {dtype}")
        bits = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
        x = bits[bits.float() <= (448 if dtype is torch.float16 else 3e38)]
        x = x[torch.isfinite(x)]
        x = torch.cat([x, x.new_zeros(-x.numel() % (t * d))]).view(-1, 1, d)
        x[::2] *= -1
        blocks = x.shape[0] // t
        cache = _random_cache(torch.Generator().manual_seed(5), blocks, 1, t, d)
        _check_write(cache, x, x.flip(0), list(range(blocks * t)), t)


@pytest.mark.parametrize("top", [448.0, 447.0, 450.0, 1.75 * 2 ** -20, 0.0, 2.0 ** -24, 65504.0])
def test_write_scale_borders(top):
    t, d = 16, 64
    cache = _random_cache(torch.Generator().manual_seed(6), 2, 2, t, d)
    for dtype in (torch.float16, torch.bfloat16):
        x = torch.zeros(3, 2, d, dtype=dtype)
        x[1, 0, 7] = top
        x[2, 1, 9] = -top
        _check_write(cache, x, x, [0, 1, 2], t)
        _check_write(cache, x, x, [21, 22, 23], t)


def test_write_strided_and_empty():
    pc = _pc()
    g = torch.Generator().manual_seed(8)
    t, kv, d = 32, 3, 64
    cache = _random_cache(g, 6, kv, t, d)
    qkv = torch.randn(40, 4 * kv, d, generator=g).bfloat16()
    dev = qkv.to(DEV)
    slots = list(range(20, 60))
    _check_write(cache, qkv[:, kv:2 * kv], qkv[:, 2 * kv:3 * kv], slots, t, (dev[:, kv:2 * kv], dev[:, 2 * kv:3 * kv]))
    odd = torch.randn(40, kv, d + 3, generator=g).bfloat16()
    dev = odd.to(DEV)
    _check_write(cache, odd[..., 1:d + 1], odd[..., 2:d + 2], slots, t, (dev[..., 1:d + 1], dev[..., 2:d + 2]))
    _check_write(cache, qkv[:0, :kv], qkv[:0, :kv], [], t)
    # a slice of every second block of a larger pool
    big = pc.PagedCache(*(x.to(DEV) for x in cache))
    half = pc.PagedCache(*(x[::2] for x in big))
    before = [x.view(torch.uint8).clone() for x in big]
    k = qkv[:, :kv].to(DEV)
    pc.write_blocks(k, k, half, _i64(list(range(40))).to(DEV))
    alone = pc.PagedCache(*(x[::2].view(torch.uint8).contiguous().view(x.dtype).to(DEV) for x in cache))
    pc.write_blocks(k, k, alone, _i64(list(range(40))).to(DEV))
    for h, a, w, was in zip(half, alone, big, before):
        assert torch.equal(h.view(torch.uint8), a.view(torch.uint8))
        assert torch.equal(w.view(torch.uint8)[1::2], was[1::2])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attend_ref(q, cache, tables, starts, lengths, window, sinks, scale):
    """(out, sum p |v| / sum p) in float64, a row at a time."""
    rows, heads, d = q.shape
    blocks, kv, t, _ = cache.k.shape
    k, v = cache.k.float().double(), cache.v.float().double().transpose(-1, -2)
    ks, vs = (2.0 ** (s.view(torch.uint8).double() - 127) for s in (cache.k_scale, cache.v_scale))
    out, mag = torch.zeros(rows, heads, d).double(), torch.zeros(rows, heads, d).double()
    for b, n in enumerate(lengths):
        for row in range(starts[b], starts[b + 1]):
            p = n - (starts[b + 1] - row)
            if n < 0 or p < 0:
                continue
            js = [j for j in range(min(p + 1, len(tables[b]) * t))
                  if 0 <= tables[b][j // t] < blocks and (not window or j > p - window or j < sinks)]
            if not js:
                continue
            js = torch.tensor(js)
            ids, off = torch.tensor(tables[b])[js // t], js % t
            kk = (k[ids, :, off] * ks[ids][..., None]).repeat_interleave(heads // kv, 1)  # [L, H, D]
            vv = (v[ids, :, off] * vs[ids][..., None]).repeat_interleave(heads // kv, 1)
            s = (kk * q[row].double()).sum(-1) * scale
            w = torch.softmax(s, 0)[..., None]
            out[row], mag[row] = (w * vv).sum(0), (w * vv.abs()).sum(0)
    return out, mag


def _attend_check(got, out, mag, dtype, top):
    h = torch.finfo(dtype).eps / 2
    tol = h * out.abs() + 3 * 2.0 ** -11 * mag + 2.0 ** -25 * top + torch.finfo(dtype).tiny * 2.0 ** -8
    got = got.double().cpu()
    assert torch.equal(got.isnan(), out.isnan())
    off = ((got - out).abs() / tol).nan_to_num(0.0)
    assert off.max() <= 1, f"error {off.max():.3f} of the tolerance"


def _attend_case(g, rng, batch, kv, group, d, t, dtype, news, most, spare=3):
    """A cache with sequences of up to ``most`` positions and rows for them."""
    lengths, starts, have = [], [0], []
    for b in range(batch):
        n = rng.choice(news)
        length = rng.choice([-1, n, n + 1, 15, 16, 17, 63, 64, 65, 255, 256, 257, rng.randrange(most + 1)])
        length = -1 if length < 0 else min(most, max(length, n))
        lengths.append(length)
        starts.append(starts[-1] + n)
        have.append(-(-max(length, 0) // t))
    ids = list(range(sum(have) + spare))
    rng.shuffle(ids)
    width = max(have) + rng.choice([1, 5])
    tables = []
    for n in have:
        tables.append(ids[:n] + [-1] * (width - n))
        ids = ids[n:]
    blocks = sum(have) + spare
    pc = _pc()

    def codes(*shape):
        return (torch.randn(shape, generator=g) * 70).clamp(-448, 448).to(F8)

    cache = pc.PagedCache(codes(blocks, kv, t, d), codes(blocks, kv, d, t),
                          *(torch.randint(127 - 9, 127 - 5, (blocks, kv), generator=g).to(torch.uint8).view(E8)
                            for _ in range(2)))
    # memory that nothing has written: NaN behind the sequences' ends, in free blocks
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    k[ids], v[ids] = 0x7F, 0xFF
    for n, r in zip(lengths, tables):
        if n > 0 and n % t:
            k[r[n // t], :, n % t:], v[r[n // t], :, :, n % t:] = 0xFF, 0x7F
    q = (torch.randn(starts[-1] + 2, kv * group, d, generator=g) * 1.5).to(dtype)
    return q, cache, tables, starts, lengths


def _attend_gpu(q, cache, tables, starts, lengths, **kw):
    pc = _pc()
    dev = pc.PagedCache(*(x.to(DEV) for x in cache))
    return pc.paged_attention(q.to(DEV), dev, torch.tensor(tables, dtype=torch.int32, device=DEV),
                              _i64(starts).to(DEV), _i64(lengths).to(DEV), **kw)


def _top(cache):
    codes = cache.v.float()
    scale = 2.0 ** (cache.v_scale.view(torch.uint8).float() - 127)
    return float((codes * scale[..., None, None]).abs().nan_to_num(0.0).max())


def _attend_compare(case, window=None, sinks=0, scale=None):
    q, cache = case[0], case[1]
    got = _attend_gpu(*case, window=window, sinks=sinks, scale=scale)
    out, mag = _attend_ref(*case, window, sinks, 1 / math.sqrt(q.shape[2]) if scale is None else scale)
    _attend_check(got, out, mag, q.dtype, _top(cache))
    return got


@pytest.mark.parametrize("seed", range(48))
def test_attention(seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    d, t = [64, 128, 256][seed % 3], [16, 32, 64, 128][seed % 4]
    group, kv = rng.choice([1, 2, 3, 4, 7, 8, 16, 20]), rng.choice([1, 2, 3])
    dtype = [torch.bfloat16, torch.float16][seed // 2 % 2]
    news = [[1], [1, 2], [1, 5, 17], [0, 1, 40, 70]][seed % 4]
    batch = rng.choice([1, 2, 5]) if group * max(news) < 500 else 1
    window = rng.choice([None, 1, 16, 100, 300])
    sinks = rng.choice([0, 1, 4, 70])
    say(f"attention seed={seed} d={d} t={t} group={group} kv={kv} {dtype} batch={batch} news={news} "
        f"window={window} sinks={sinks}")
    case = _attend_case(g, rng, batch, kv, group, d, t, dtype, news, 1500)
    _attend_compare(case, window, sinks)


@pytest.mark.parametrize("d,t,n,length", [(128, 64, 1, 9000), (64, 16, 3, 5000), (256, 128, 1, 5000),
                                          (128, 32, 16, 3000), (128, 64, 200, 700), (64, 64, 300, 300)])
def test_attention_long(d, t, n, length):
    """Sequences that are divided between workgroups, short ones beside them."""
    say(f"attention d={d} t={t} n={n} length={length}")
    rng, g = random.Random(3), torch.Generator().manual_seed(3)
    pc = _pc()
    q, cache, tables, starts, lengths = _attend_case(g, rng, 1, 2, 4, d, t, torch.bfloat16, [n], length, 2)
    while lengths != [length]:
        q, cache, tables, starts, lengths = _attend_case(g, rng, 1, 2, 4, d, t, torch.bfloat16, [n], length, 2)
        if lengths[0] > length // 2:
            break
    for window, sinks in ((None, 0), (length // 3, 5)):
        _attend_compare((q, cache, tables, starts, lengths), window, sinks)


def test_attention_batch_of_many():
    """More sequences than a wave has lanes, most of them short, some empty."""
    say("attention batch of 150")
    rng, g = random.Random(9), torch.Generator().manual_seed(9)
    _attend_compare(_attend_case(g, rng, 150, 2, 4, 64, 16, torch.float16, [0, 1, 1, 2], 300))


def test_attention_tables_with_holes():
    """Positions whose block is none of the cache's are not seen; a row may see nothing."""
    say("attention tables with holes")
    rng, g = random.Random(10), torch.Generator().manual_seed(10)
    q, cache, tables, starts, lengths = _attend_case(g, rng, 4, 2, 3, 128, 16, torch.bfloat16, [1, 20], 400)
    lengths = [max(n, starts[b + 1] - starts[b]) for b, n in enumerate(lengths)]
    width = len(tables[0])
    for r in tables:
        for j in range(0, width, 2):
            r[j] = rng.choice([-1, -(1 << 31), cache.k.shape[0], (1 << 31) - 1])
    tables[1] = [-1] * width
    got = _attend_compare((q, cache, tables, starts, lengths))
    assert not got[starts[1]:starts[2]].any()
    _attend_compare((q, cache, tables, starts, lengths), 20, 3)
    # lengths past the table's end
    _attend_compare((q, cache, tables, starts, [n + 1000 for n in lengths]))


@pytest.mark.parametrize("group,n", [(4, 1), (4, 30), (8, 100)])
def test_attention_values_that_are_not_finite(group, n):
    """NaN keys and values reach the rows that see them and no others: later tokens of
    a chunk, and what a window has left behind."""
    say(f"attention NaN codes group={group} n={n}")
    rng, g = random.Random(11), torch.Generator().manual_seed(11)
    pc = _pc()
    t, length = 32, 333
    q, cache, tables, starts, lengths = _attend_case(g, rng, 1, 2, group, 128, t, torch.bfloat16, [n], length)
    while lengths[0] < 300:
        q, cache, tables, starts, lengths = _attend_case(g, rng, 1, 2, group, 128, t, torch.bfloat16, [n], length)
    end = lengths[0]
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    def at(j):
        return tables[0][j // t], j % t
    b, o = at(end - 1 - n // 2)
    v[b, 0, 5, o] = 0x7F           # a token within the chunk: one dimension of one head
    b, o = at(100)
    v[b, 1, :, o] = 0xFF           # behind a window
    b, o = at(2)
    k[b, 0, 9, o] = 0x7F           # a first position
    for window, sinks in ((None, 0), (64, 0), (64, 2), (64, 3), (150, 1)):
        _attend_compare((q, cache, tables, starts, lengths), window, sinks)
    # queries that are not finite
    q[0, 0, 0], q[min(n, 2) - 1, 1, 3] = float("inf"), NAN
    got = _attend_gpu(q, cache, tables, starts, lengths, window=64)
    out, mag = _attend_ref(q, cache, tables, starts, lengths, 64, 0, 1 / math.sqrt(128))
    clean = ~out.isnan().any(-1)
    assert torch.equal(got.isnan().any(-1).cpu(), ~clean)
    _attend_check(got[clean.to(DEV)], out[clean], mag[clean], q.dtype, _top(cache))


def test_attention_scales_far_apart():
    """Blocks of zeros, of tiny and of large values in one sequence."""
    rng, g = random.Random(12), torch.Generator().manual_seed(12)
    for dtype, low, high in ((torch.bfloat16, -60, 30), (torch.float16, -20, 4)):
        q, cache, tables, starts, lengths = _attend_case(g, rng, 3, 2, 4, 128, 16, dtype, [1, 9], 600)
        lengths = [max(n, 200) if n >= 0 else n for n in lengths]
        case = _attend_case(g, rng, 3, 2, 4, 128, 16, dtype, [1, 9], 600)
        q, cache, tables, starts, lengths = case
        blocks = cache.k.shape[0]
        cache.v_scale.view(torch.uint8).copy_(torch.randint(127 + low, 127 + high, (blocks, 2), generator=g))
        cache.v.view(torch.uint8)[::3] = 0
        cache.v_scale.view(torch.uint8)[::3] = 127 + LEAST
        say(f"attention scales {low}..{high}")
        _attend_compare(case)


def test_attention_peaked_and_flat():
    """A scale of 0 (all alike) and one so large that single keys carry a row."""
    say("attention scale 0 and 20")
    rng, g = random.Random(13), torch.Generator().manual_seed(13)
    case = _attend_case(g, rng, 3, 2, 4, 64, 32, torch.float16, [1, 9], 700)
    _attend_compare(case, scale=0.0)
    case = (case[0] * 0.25, *case[1:])
    _attend_compare(case, 200, 4, scale=1.0)


def test_attention_strided_queries_and_empty_batches():
    pc = _pc()
    rng, g = random.Random(14), torch.Generator().manual_seed(14)
    q, cache, tables, starts, lengths = _attend_case(g, rng, 2, 2, 4, 64, 16, torch.bfloat16, [1, 3], 300)
    say("attention strided queries")
    dev = pc.PagedCache(*(x.to(DEV) for x in cache))
    rest = (dev, torch.tensor(tables, dtype=torch.int32, device=DEV), _i64(starts).to(DEV), _i64(lengths).to(DEV))
    want = pc.paged_attention(q.to(DEV), *rest)
    wide = torch.randn(q.shape[0], 12, 64, device=DEV).bfloat16()
    wide[:, 2:10] = q.to(DEV)
    assert torch.equal(pc.paged_attention(wide[:, 2:10], *rest), want)
    odd = torch.randn(q.shape[0], 8, 65, device=DEV).bfloat16()
    odd[..., 1:] = q.to(DEV)
    assert torch.equal(pc.paged_attention(odd[..., 1:], *rest), want)
    tab = torch.full((2, 2 * len(tables[0])), -1, dtype=torch.int32, device=DEV)
    tab[:, ::2] = rest[1]
    assert torch.equal(pc.paged_attention(q.to(DEV), dev, tab[:, ::2], *rest[2:]), want)
    assert not pc.paged_attention(q.to(DEV), dev, rest[1], torch.zeros_like(rest[2]), rest[3]).any()
    # a window and first positions past everything
    assert torch.equal(pc.paged_attention(q.to(DEV), *rest, window=1 << 70, sinks=1 << 70), want)
    # every second block of a larger pool, whose others hold NaN
    def wide(x):
        big = torch.full((2 * x.shape[0], *x.shape[1:]), 0x7F, dtype=torch.uint8, device=DEV).view(x.dtype)
        big.view(torch.uint8)[::2] = x.view(torch.uint8)
        return big[::2]
    assert torch.equal(pc.paged_attention(q.to(DEV), pc.PagedCache(*(wide(x) for x in dev)), *rest[1:]), want)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_rows_outside_all_sequences(n):
    """Rows before the first sequence's, too, and batches of which nothing is left."""
    say(f"attention rows outside n={n}")
    rng, g = random.Random(19), torch.Generator().manual_seed(19)
    q, cache, tables, starts, lengths = _attend_case(g, rng, 3, 2, 4, 64, 16, torch.float16, [n], 400)
    lengths = [max(x, n) for x in lengths]
    rows = starts[-1] + 9
    q = torch.randn(rows, 8, 64, generator=g).half()
    got = _attend_compare((q, cache, tables, [s + 5 for s in starts], lengths))
    assert not got[:5].any() and not got[-4:].any() and got[5:-4].any()
    assert not _attend_gpu(q, cache, tables, starts, [-1, -1, -1]).any()
    # more rows than positions: those before position 0 see nothing
    _attend_compare((q, cache, tables, starts, [min(x, 1 + n // 2) for x in lengths]), 3, 1)


def test_attention_and_write_past_32_bits():
    """A pool whose codes pass 2^32 bytes: the last blocks hold a sequence."""
    say("pool past 2^32 bytes")
    pc = _pc()
    kv, t, d = 8, 128, 256
    blocks = (1 << 32) // (kv * t * d) + 40
    cache = pc.PagedCache(torch.zeros(blocks, kv, t, d, dtype=torch.uint8, device=DEV).view(F8),
                          torch.zeros(blocks, kv, d, t, dtype=torch.uint8, device=DEV).view(F8),
                          *(torch.full((blocks, kv), 127, dtype=torch.uint8, device=DEV).view(E8) for _ in range(2)))
    small = pc.new_cache(40, kv, t, d, DEV)
    g = torch.Generator(device=DEV).manual_seed(15)
    n = 5 * t + 17
    k, v = (torch.randn(n, kv, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    q = torch.randn(3, 2 * kv, d, generator=g, device=DEV).bfloat16()
    got = []
    for c, first in ((small, 0), (cache, blocks - 40)):
        ids = torch.arange(5, -1, -1, device=DEV) * 7 + first
        slots = ids[torch.arange(n, device=DEV) // t] * t + torch.arange(n, device=DEV) % t
        pc.write_blocks(k, v, c, slots)
        got.append(pc.paged_attention(q, c, ids.int()[None], _i64([0, 3]).to(DEV), _i64([n]).to(DEV)))
    assert torch.equal(got[0], got[1]) and got[0].any()
    assert torch.equal(cache.k[blocks - 40:].view(torch.uint8), small.k.view(torch.uint8))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_steps_together():
    """Prompts in chunks beside decodes, sequences that finish and start, drafts taken
    back: each step's attention over what the cache stands for, in float64."""
    pc = _pc()
    t, kv, group, d, width, rows = 16, 2, 4, 64, 24, 96
    g = torch.Generator().manual_seed(16)
    rng = random.Random(16)
    batch, blocks = 5, 60
    cache = pc.PagedCache(*(x.to(DEV) for x in _random_cache(g, blocks, kv, t, d)))
    free, count = torch.arange(blocks, dtype=torch.int32, device=DEV), _i64([blocks]).to(DEV)
    tables = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    lengths = _i64([0, 0, -1, 0, 0]).to(DEV)
    written = [[] for _ in range(batch)]  # what each sequence's cache was given
    for step in range(14):
        counts = _i64([rng.choice([1, 1, 3, 30, 0]) for _ in range(batch)])
        plan = pc.plan_step(lengths, counts.to(DEV), tables, free, count, rows, t)
        k, v = (torch.randn(rows, kv, d, generator=g).bfloat16() for _ in range(2))
        q = torch.randn(rows, kv * group, d, generator=g).bfloat16()
        pc.write_blocks(k.to(DEV), v.to(DEV), cache, plan.slots)
        o = pc.paged_attention(q.to(DEV), cache, tables, plan.starts, plan.lengths, 100, 4)
        say(f"step {step}: lengths {lengths.tolist()} counts {counts.tolist()}")
        host = pc.PagedCache(*(x.cpu() for x in cache))
        out, mag = _attend_ref(q, host, tables.tolist(), plan.starts.tolist(), plan.lengths.tolist(), 100, 4,
                               1 / math.sqrt(d))
        _attend_check(o, out, mag, q.dtype, 30.0)
        starts, after = plan.starts.tolist(), plan.lengths.tolist()
        ks, vs = (2.0 ** (s.view(torch.uint8).double() - 127) for s in (host.k_scale, host.v_scale))
        for b in range(batch):
            if after[b] >= 0:
                written[b] = written[b][:lengths[b].item()]
                written[b] += [(k[r], v[r]) for r in range(starts[b], starts[b + 1])]
            # a code is within 1/16 of its value, or 2^-10 of the block's scale, once or
            # twice (a scale that grew): 0.14 of it and 2^-9 of the scale
            for j, (kk, vv) in enumerate(written[b]):
                block, off = tables[b, j // t].item(), j % t
                for codes, s, x in ((host.k[block, :, off].float(), ks, kk), (host.v[block, :, :, off].float(), vs, vv)):
                    err = (codes.double() * s[block][:, None] - x.double()).abs()
                    assert (err <= 0.14 * x.double().abs() + 2.0 ** -9 * s[block][:, None]).all()
        lengths = torch.where(plan.lengths >= 0, plan.lengths, lengths)
        if step % 3 == 1:  # the last tokens were drafts
            lengths = (lengths - 2).clamp(min=-1)
        keep = lengths.clone()
        if step % 4 == 3:  # one is done, another takes its place
            done = rng.randrange(batch)
            keep[done], lengths[done] = 0, 0
            written[done] = []
        pc.release_blocks(tables, keep, free, count, t)
        owned = tables[tables >= 0].tolist() + free[:count.item()].tolist()
        assert sorted(owned) == list(range(blocks))


def test_captured_step():
    """A step replayed from a graph serves other lengths, counts and tokens; eager work
    on the same pool runs between the replays."""
    pc = _pc()
    t, kv, group, d, width, rows, batch, blocks = 32, 2, 4, 128, 40, 70, 4, 120
    g = torch.Generator(device=DEV).manual_seed(17)

    def pool():
        return (pc.new_cache(blocks, kv, t, d, DEV), torch.full((batch, width), -1, dtype=torch.int32, device=DEV),
                torch.arange(blocks, dtype=torch.int32, device=DEV), _i64([blocks]).to(DEV),
                _i64([0] * batch).to(DEV))

    def step(state, counts, k, v, q):
        cache, tables, free, count, lengths = state
        plan = pc.plan_step(lengths, counts, tables, free, count, rows, t)
        pc.write_blocks(k, v, cache, plan.slots)
        o = pc.paged_attention(q, cache, tables, plan.starts, plan.lengths, 300, 4)
        pc.release_blocks(tables, torch.where(plan.lengths > 900, 0, -1), free, count, t)
        lengths.copy_(torch.where(plan.lengths > 900, 0, torch.where(plan.lengths >= 0, plan.lengths, lengths)))
        return o

    counts = _i64([1] * batch).to(DEV)
    k, v = (torch.zeros(rows, kv, d, device=DEV).bfloat16() for _ in range(2))
    q = torch.zeros(rows, kv * group, d, device=DEV).bfloat16()
    graphed, eager = pool(), pool()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(pool(), counts, k, v, q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            o = step(graphed, counts, k, v, q)
    torch.cuda.synchronize()
    for i in range(24):
        n = [[1, 1, 1, 1], [60, 1, 0, 5], [1, 1, 60, 1], [0, 65, 1, 2]][i % 4]
        counts.copy_(_i64(n))
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        graph.replay()
        want = step(eager, counts, k, v, q)
        say(f"replay {i}: lengths {eager[4].tolist()}")
        assert torch.equal(o, want)
        for a, b in zip(graphed[1:], eager[1:]):
            assert torch.equal(a, b)
        for a, b in zip(graphed[0], eager[0]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_other_stream_and_two_at_once():
    """Calls on two streams at once give what they give alone."""
    pc = _pc()
    rng, g = random.Random(18), torch.Generator().manual_seed(18)
    cases = [_attend_case(g, rng, 3, 2, 4, 128, 64, torch.bfloat16, [1, 6], 3000) for _ in range(2)]
    dev = [(c[0].to(DEV), pc.PagedCache(*(x.to(DEV) for x in c[1])), torch.tensor(c[2], dtype=torch.int32, device=DEV),
            _i64(c[3]).to(DEV), _i64(c[4]).to(DEV)) for c in cases]
    want = [pc.paged_attention(*c) for c in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    for _ in range(10):
        got = []
        for s, c in zip(streams, dev):
            with torch.cuda.stream(s):
                got.append(pc.paged_attention(*c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_inference_mode_versions_and_gradients():
    pc = _pc()
    cache = pc.new_cache(4, 2, 16, 64, DEV)
    k = torch.randn(3, 2, 64, device=DEV).bfloat16()
    slots = _i64([0, 1, 2]).to(DEV)
    before = [x._version for x in cache]
    pc.write_blocks(k, k, cache, slots)
    assert all(x._version > n for x, n in zip(cache, before))
    with torch.inference_mode():
        pc.write_blocks(k, k, pc.new_cache(4, 2, 16, 64, DEV), slots)
    with pytest.raises(RuntimeError, match="no backward pass"):
        pc.write_blocks(k.clone().requires_grad_(), k, cache, slots)
    with pytest.raises(RuntimeError, match="no backward pass"):
        pc.paged_attention(k.clone().requires_grad_(), cache, torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                           _i64([0, 3]).to(DEV), _i64([3]).to(DEV))
    with pytest.raises(RuntimeError, match="GPU only|different devices"):
        pc.write_blocks(k, k, cache, slots.cpu())
