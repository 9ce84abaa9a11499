"""GPU tests of the attention of drafted tokens with fp16 caches where one key has
most of the weight, against float64.

Tolerance. As for the other cases (half a step of the result; each probability
rounded to fp16 in the sum of the values and in the sum that divides them, 2^-10 of
A = sum p |v| / sum p; scores in fp32, 2^-12 A), but for probabilities below fp16's
normal range: the largest is held at 2^7 or more, the absolute rounding there is
2^-25, so each is off by at most 2^-32 of the largest, which is no more than the sum
that divides: 2^-32 sum |v|."""

import pytest
import torch

import test_gpu_tree_decode as base
from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu


def _check(got, want, what):
    out, size, total = want
    f = torch.finfo(torch.float16)
    err = (got.double().cpu() - out).abs()
    tol = (f.eps / 2 * out.abs() + (f.eps + 2.0 ** -12) * size + 2.0 ** -32 * total
           + f.smallest_normal * f.eps / 2)
    bad = ~(err <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} off, worst {float(err[bad].max()):.3e} "
                                 f"of {float(out[bad].abs().max()):.3e}")


def _case(length, n, heads, dim, gap, at):
    """Scores of +-1/2 but for the key at ``at``, ``gap`` above them, whose value is 0."""
    g = torch.Generator().manual_seed(length + dim)
    q, k, v, lengths, masks = base._attention_case(3, [length], n, heads, 1, dim, torch.float16, "row")
    q = torch.randn(q.shape, generator=g)
    q[..., 0] = 8.0
    k = torch.randn(k.shape, generator=g) * 0.5
    k[..., 0] = 0.0
    k[0, 0, at] = 0.0
    k[0, 0, at, 0] = gap * dim ** 0.5 / 8.0
    v = torch.randn(v.shape, generator=g) * 0.5 + 1.0
    v[0, 0, at] = 0.0
    return q.half(), k.half(), v.half(), lengths, masks


def _shared(case, layout, batch):
    """The case for ``batch`` sequences over one cache: so many that a workgroup goes
    through a sequence's tiles one after the other instead of taking a few of them."""
    q, k, v, lengths, masks = case
    kd, vd = (base._to_cache(t, y).expand(batch, -1, -1, -1) for t, y in ((k, layout), (v, "row")))
    return base._td().tree_attention(q.to(DEV).expand(batch, -1, -1, -1).contiguous(), kd, vd,
                                     lengths.expand(batch).to(DEV), masks[0].to(DEV))


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("n,heads,dim,length", [
    (4, 2, 64, 9000), (6, 4, 128, 9000), (12, 4, 128, 32000), (64, 4, 64, 3000), (64, 4, 128, 3000),
    (5, 1, 256, 9000), (33, 1, 256, 9000), (64, 2, 256, 3000)])
@pytest.mark.parametrize("gap", [13.0, 17.0, 18.0])
def test_one_key_far_above_the_others(layout, n, heads, dim, length, gap):
    say(f"attention fp16 sink {layout} n={n} heads={heads} dim={dim} length={length} gap={gap}")
    case = _case(length, n, heads, dim, gap, 0)
    got = _shared(case, layout, 600 if dim < 256 else 300)
    want = base._attend_ref(*case, dim ** -0.5)
    _check(got, [t.expand_as(got) for t in want], f"gap {gap}")


@pytest.mark.parametrize("gap", [3.0, 5.5, 6.0, 17.0])
@pytest.mark.parametrize("at", [70, 2500])
@pytest.mark.parametrize("bad", [False, True])
def test_a_key_that_comes_later(gap, at, bad):
    """The largest score where the exponents' base may not have followed it (factors up
    to 2^8), once and many times; ``bad``: with a drafted value that is not finite and
    that most nodes do not see."""
    say(f"attention fp16 later key gap={gap} at={at} bad={bad}")
    n, dim = 6, 128
    q, k, v, lengths, masks = _case(4001, n, 4, dim, gap, at)
    k[0, 0, at:at + 60] = k[0, 0, at].clone()
    v[0, 0, at:at + 60:2] = 0.0
    want = base._attend_ref(q, k, v, lengths, masks, dim ** -0.5)
    rows = slice(None)
    if bad:
        masks[0, 1:] &= ~2
        masks[0, 1] |= 2
        want = base._attend_ref(q, k, v, lengths, masks, dim ** -0.5)
        v[0, 0, 4002] = float("inf")
        rows = [i for i in range(n) if i != 1]
    got = _shared((q, k, v, lengths, masks), "row", 600)
    _check(got[:, rows], [t[:, rows].expand_as(got[:, rows]) for t in want], f"gap {gap}")
