"""GPU tests of paged attention where blocks' scales lie far apart: what a row does not see
has no effect on it, and what it sees counts by its own weight and size, whatever other
rows, other sequences and free blocks hold. Against float64 on the CPU.

Tolerance of one result, from what its own row sees alone. A = sum p |v| / sum p: the
probabilities' rounding to fp16, 2^-11 of itself, and that of the scores, fp32 sums of
products below 2^-11 in the exponent (as test_gpu_paged_cache counts it), in the sum of
values and in the sum that divides: 3 * 2^-11 A. What multiplies a code, probability times
scale, is rounded to fp16 in units of the row's largest such product T, at most one power of
two above it and lifted by 2^7: half the smallest subnormal, 2^-25, is 2^-31 T, for each
code once: 2^-31 T sum |code|. The result is rounded once: half a step, h = finfo.eps / 2."""

import math

import pytest
import torch

from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _pc():
    from polarengine_vllm.kernels import paged_cache
    return paged_cache


def _i64(x):
    return torch.tensor(x, dtype=torch.int64)


def _case(seed, batch, kv, group, d, t, dtype, news, lengths, spare=2, extra=0):
    """A cache with sequences of ``lengths`` whose last ``news`` rows are asked for;
    ``extra`` more blocks of each table behind its sequence's end. Scales of 2^-9..2^-6."""
    g = torch.Generator().manual_seed(seed)
    have = [-(-n // t) + extra for n in lengths]
    blocks = sum(have) + spare
    ids = torch.randperm(blocks, generator=g).tolist()
    width = max(have) + 1
    tables, starts = [], [0]
    for n, new in zip(have, news):
        tables.append(ids[:n] + [-1] * (width - n))
        ids = ids[n:]
        starts.append(starts[-1] + new)

    def codes(*shape):
        return (torch.randn(shape, generator=g) * 70).clamp(-448, 448).to(F8)

    cache = _pc().PagedCache(codes(blocks, kv, t, d), codes(blocks, kv, d, t),
                             *(torch.randint(127 - 9, 127 - 5, (blocks, kv), generator=g).to(torch.uint8).view(E8)
                               for _ in range(2)))
    q = (torch.randn(starts[-1], kv * group, d, generator=g) * 1.5).to(dtype)
    return q, cache, tables, starts, list(lengths)


def _ref(q, cache, tables, starts, lengths, window, sinks, scale):
    """(out, A, T sum |code|) of each row, head and dimension in float64."""
    rows, heads, d = q.shape
    kv, t = cache.k.shape[1], cache.k.shape[2]
    group = heads // kv
    codes = [x.float().double().nan_to_num(0.0) for x in (cache.k, cache.v.transpose(-1, -2))]
    exps = [s.view(torch.uint8).double() - 127 for s in (cache.k_scale, cache.v_scale)]
    out = torch.zeros(rows, heads, d).double()
    mag, unit = torch.zeros_like(out), torch.zeros_like(out)
    for b, n in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        if hi == lo:
            continue
        js = torch.arange(n)
        ids, off = torch.tensor(tables[b])[js // t], js % t
        k = (codes[0][ids, :, off] * (2.0 ** exps[0][ids])[..., None]).transpose(0, 1)  # [kv, n, d]
        vc, ve = codes[1][ids, :, off].transpose(0, 1), exps[1][ids].t()
        p = torch.arange(n - (hi - lo), n)[:, None]
        seen = js <= p
        if window:
            seen &= (js > p - window) | (js < sinks)
        for h in range(heads):
            s = (q[lo:hi, h].double() @ k[h // group].t()) * scale
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            x = w * 2.0 ** ve[h // group]
            out[lo:hi, h], mag[lo:hi, h] = x @ vc[h // group], x @ vc[h // group].abs()
            unit[lo:hi, h] = x.amax(-1, keepdim=True) * (seen.double() @ vc[h // group].abs())
    return out, mag, unit


def _gpu(q, cache, tables, starts, lengths, **kw):
    dev = _pc().PagedCache(*(x.to(DEV) for x in cache))
    return _pc().paged_attention(q.to(DEV), dev, torch.tensor(tables, dtype=torch.int32, device=DEV),
                                 _i64(starts).to(DEV), _i64(lengths).to(DEV), **kw).double().cpu()


def _compare(case, window=None, sinks=0, scale=None):
    q = case[0]
    got = _gpu(*case, window=window, sinks=sinks, scale=scale)
    out, mag, unit = _ref(*case, window, sinks, 1 / math.sqrt(q.shape[2]) if scale is None else scale)
    info = torch.finfo(q.dtype)
    tol = info.eps / 2 * out.abs() + 3 * 2.0 ** -11 * mag + 2.0 ** -31 * unit + info.tiny * info.eps
    assert bool(torch.isfinite(got).all())
    off = (got - out).abs() / tol
    assert off.max() <= 1, f"error {off.max():.3f} of the tolerance"
    return got


def _bytes(scale):
    return scale.view(torch.uint8)


# (rows of a sequence, group, head size): few rows and chunks, every kernel
FORMS = [(1, 4, 64), (1, 8, 128), (3, 2, 256), (9, 4, 128), (12, 4, 64), (40, 4, 64), (40, 8, 128), (40, 8, 256)]


@pytest.mark.parametrize("new,group,d", FORMS)
@pytest.mark.parametrize("byte", [1, 160, 200, 255])
def test_scales_behind_the_end(new, group, d, byte):
    """Blocks that a table names already, and that nothing has written yet: their scales
    change nothing, bit for bit."""
    say(f"scales behind the end {new} x {group} x {d} byte {byte}")
    case = _case(d + new, 2, 2, group, d, 16, torch.bfloat16, [new, new], [100, 333], extra=4)
    want = _compare(case)
    q, cache, tables, starts, lengths = case
    for b, n in enumerate(lengths):
        behind = [i for i in tables[b][-(-n // 16):] if i >= 0]
        assert len(behind) == 4
        for s in (cache.k_scale, cache.v_scale):
            _bytes(s)[behind] = byte
        cache.k.view(torch.uint8)[behind], cache.v.view(torch.uint8)[behind] = 0x7F, 0xFF
    assert torch.equal(_compare(case), want)


@pytest.mark.parametrize("new,group,d", FORMS)
def test_scales_behind_a_window(new, group, d):
    """Blocks between the first positions and every row's window."""
    window, sinks = 70, 5
    for dtype in (torch.bfloat16, torch.float16):
        say(f"scales behind a window {new} x {group} x {d} {dtype}")
        case = _case(d * new, 2, 2, group, d, 16, dtype, [new, new], [300, 411])
        want = _compare(case, window, sinks)
        q, cache, tables, starts, lengths = case
        for b, n in enumerate(lengths):
            hidden = tables[b][1:(n - new + 1 - window) // 16]
            assert len(hidden) > 8
            _bytes(cache.v_scale)[hidden] = torch.randint(200, 250, (len(hidden), 2)).to(torch.uint8)
            _bytes(cache.k_scale)[hidden] = 160
        assert torch.equal(_compare(case, window, sinks), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,group,d", [f for f in FORMS if f[0] > 2])
def test_scales_of_later_tokens(new, group, d, dtype):
    """Rows of a chunk before one whose block's values are 2^40 times as large: each is
    held to what it sees, and equals the row of a chunk that ends there."""
    say(f"scales of later tokens {new} x {group} x {d} {dtype}")
    t, length = 16, 250
    case = _case(d + 3 * new, 1, 2, group, d, t, dtype, [new], [length])
    q, cache, tables, starts, lengths = case
    _bytes(cache.v_scale).sub_(14 if dtype is torch.float16 else 40)
    last = tables[0][15]  # positions from 240 on, behind others of one step of 64
    _bytes(cache.v_scale)[last] += 24 if dtype is torch.float16 else 60
    if new <= 10:  # all rows would see it: the first is put before it
        case = q, cache, tables, starts, [239 + new]
    _compare(case)
    _compare(case, 64, 3)


@pytest.mark.parametrize("new,group,d", FORMS)
@pytest.mark.parametrize("scale", [None, 0.0, 2.0])
def test_scales_of_any_size(new, group, d, scale):
    """Blocks of every scale from 2^-100 up, some of them zeros, at flat and at peaked
    weights: a block without weight costs those with weight nothing."""
    for dtype, low, high in ((torch.bfloat16, 27, 200), (torch.float16, 100, 130)):
        say(f"scales of any size {new} x {group} x {d} {dtype} scale {scale}")
        case = _case(7 * d + new, 3, 2, group, d, 16, dtype, [new] * 3, [60, 230, 700])
        cache = case[1]
        g = torch.Generator().manual_seed(new)
        blocks = cache.k.shape[0]
        _bytes(cache.v_scale).copy_(torch.randint(low, high, (blocks, 2), generator=g))
        cache.v.view(torch.uint8)[::5] = 0
        _bytes(cache.v_scale)[::5] = 27
        if scale == 2.0:  # |score| stays below 40
            case = (case[0] / 16 / math.sqrt(d / 64), *case[1:])
        _compare(case, scale=scale)
        _compare(case, 100, 20, scale=scale)


@pytest.mark.parametrize("new,group,d", FORMS)
def test_scores_past_whole_numbers(new, group, d):
    """Scores so large that fp32 holds no fractions of them: one key carries each row, and
    the result is its value, whatever its block's scale."""
    say(f"scores past whole numbers {new} x {group} x {d}")
    case = _case(d - new, 2, 1, group, d, 16, torch.bfloat16, [new, new], [400, 150])
    q, cache, tables, starts, lengths = case
    g = torch.Generator().manual_seed(5)
    _bytes(cache.v_scale).copy_(torch.randint(60, 190, (cache.k.shape[0], 1), generator=g))
    # keys of one value each, all different from the next by a sixteenth at least, the
    # largest among them (448) once a sequence
    for b, n in enumerate(lengths):
        level = torch.randint(1, 29, (n,), generator=g) * 8.0
        level[int(torch.randint(0, n - new, (1,), generator=g))] = 448.0
        for j in range(n):
            cache.k[tables[b][j // 16], 0, j % 16] = level[j].to(F8)
    _bytes(cache.k_scale)[:] = 127
    q = torch.full_like(q, 2.0 ** 20)
    _compare((q, cache, tables, starts, lengths), scale=1.0)


@pytest.mark.parametrize("d,t,new,length", [(64, 16, 3, 5000), (128, 64, 1, 9000), (256, 128, 1, 5000), (128, 32, 16, 4100),
                                            (128, 64, 200, 700), (64, 64, 300, 300), (256, 16, 100, 2000),
                                            (64, 16, 64, 9000)])
def test_long_sequences(d, t, new, length):
    """Sequences of just this length, divided between workgroups, one a quarter as long
    beside it, with scales far apart."""
    say(f"long sequences d={d} t={t} new={new} length={length}")
    short = max(new, length // 4)
    case = _case(length, 2, 2, 4, d, t, torch.bfloat16, [new, min(new, short)], [length, short])
    _bytes(case[1].v_scale).copy_(torch.randint(60, 160, case[1].v_scale.shape, generator=torch.Generator().manual_seed(1)))
    _compare(case)
    _compare(case, length // 3, 5)


@pytest.mark.parametrize("new,group,d", FORMS)
def test_smallest_scales(new, group, d):
    """Scales that no write gives, down to the type's smallest."""
    say(f"smallest scales {new} x {group} x {d}")
    for length in (70, 900):
        case = _case(d * 2 + new, 1, 2, group, d, 16, torch.bfloat16, [new], [length])
        scale = _bytes(case[1].v_scale)
        for low, high in ((1, 2), (1, 27), (9, 14)):
            scale.copy_(torch.randint(low, high, scale.shape, generator=torch.Generator().manual_seed(low)))
            _compare(case)


@pytest.mark.parametrize("d,t,new,group,length", [(64, 128, 1, 4, 40000), (128, 64, 2, 8, 20000), (256, 128, 1, 2, 17000),
                                                  (64, 64, 40, 8, 9000), (128, 128, 50, 8, 6000)])
def test_parts_past_a_wave(d, t, new, group, length):
    """One KV head, so that a row block is divided into more parts than a wave has lanes."""
    say(f"parts past a wave d={d} new={new} length={length}")
    case = _case(length, 1, 1, group, d, t, torch.bfloat16, [new], [length])
    _compare(case)
    scale = _bytes(case[1].v_scale)
    scale.copy_(torch.randint(60, 160, scale.shape, generator=torch.Generator().manual_seed(2)))
    _compare(case)
    _compare(case, length - 700, 9)
