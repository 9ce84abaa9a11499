"""GPU tests of kernels.logprobs where logits are ruled out: a NaN logit stands for -inf,
in the given token, in ranks and among the likeliest alike. What a row with NaN answers has
to equal, bit for bit, what the same row with -inf in their place answers, which is held to
float64 with the tolerances of test_gpu_logprobs."""

import math

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_logprobs import _check, _lp

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# quiet and signalling NaN of either sign
NANS = {torch.float32: (torch.int32, [0x7FC00000, 0x7F800001, -0x400000, -0x7FFFFF]),
        torch.bfloat16: (torch.int16, [0x7FC0, 0x7F81, -0x40, -0x7F]),
        torch.float16: (torch.int16, [0x7E00, 0x7C01, -0x200, -0x3FF])}


def _case(rows, vocab, dtype, seed, finite):
    """Rows with ``finite`` finite logits, the others NaN (all kinds) and -inf by turns;
    one in four rows has finite logits everywhere but at some NaN."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    out = torch.rand(rows, vocab, generator=g)
    keep = out.argsort(1).argsort(1) < finite
    keep[::4] = out[::4] < 0.8
    kind = torch.randint(0, 5, (rows, vocab), generator=g)
    ints, nans = NANS[dtype]
    bits = torch.tensor(nans, dtype=ints).view(dtype)
    x = torch.where(keep, x, torch.where(kind == 4, -math.inf, bits[kind.clamp(max=3)]))
    return x, x.isnan()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 40001, 64), (3, 1, 1), (5, 37, 37), (9, 999, 64), (40, 12345, 20),
                                            (1500, 300, 10), (2, 100003, 0)])
def test_nan_counts_as_ruled_out(rows, vocab, top, dtype):
    say(f"ruled out {dtype} {rows} x {vocab} top {top}")
    x, nan = _case(rows, vocab, dtype, rows + vocab, max(1, top // 2))
    if vocab == 1:
        x, nan = torch.zeros(rows, 1, dtype=dtype), torch.zeros(rows, 1, dtype=torch.bool)
    clean = torch.where(nan, -math.inf, x)
    g = torch.Generator().manual_seed(7)
    for pick in range(3):
        # a token whose logit is NaN, one whose logit is -inf behind NaN, any
        of = [nan, (clean == -math.inf) & ~nan, torch.ones_like(nan)][pick]
        score = torch.where(of, torch.rand(rows, vocab, generator=g), -1.0)
        tokens = score.argmax(1)
        got = _lp().token_logprobs(x.to(DEV), tokens.to(DEV), top)
        want = _check(clean.to(DEV), tokens.to(DEV), top)
        for name, a, b in zip(got._fields, got, want):
            assert torch.equal(a, b), name
        at = nan.gather(1, tokens[:, None])[:, 0]
        assert bool((got.logprob.cpu()[at] == -math.inf).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_past_the_finite_logits(dtype):
    """Ruled-out tokens follow the finite ones, by number, whether NaN or -inf."""
    x = torch.full((2, 500), float("nan"), dtype=dtype)
    x[:, 1::2] = -math.inf
    x[0, 300], x[0, 7], x[1, 499] = 2.0, 1.0, 0.5
    out = _lp().token_logprobs(x.to(DEV), torch.tensor([4, 3], device=DEV), 6)
    assert out.top_tokens.tolist() == [[300, 7, 0, 1, 2, 3], [499, 0, 1, 2, 3, 4]]
    assert out.rank.tolist() == [6, 4] and out.logprob.tolist() == [-math.inf, -math.inf]
    assert bool((out.top_logprobs[0, 2:] == -math.inf).all())
