"""GPU tests of kernels.logprobs with finite logits at both ends of their type: values
whose differences pass fp32's range have a distribution like others."""

import math

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_logprobs import _lp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 60001), (3, 9), (2, 4099), (1500, 600)])
def test_differences_past_the_range(rows, vocab, dtype):
    """The lowest value everywhere, then two or three equal largest ones: the distribution
    is theirs alone, log probability -log n and entropy log n (2^-16, as the other tests
    have it, and half a step)."""
    say(f"extremes {dtype} {rows} x {vocab}")
    info = torch.finfo(dtype)
    x = torch.full((rows, vocab), info.min, dtype=dtype)
    at = [vocab - 1, vocab // 2, vocab // 3]
    n = torch.tensor([2 + r % 2 for r in range(rows)])
    for r in range(rows):
        x[r, at[:int(n[r])]] = info.max
    tokens = torch.full((rows,), at[1])
    out = _lp().token_logprobs(x.to(DEV), tokens.to(DEV), 2)
    want = n.double().log()
    tol = 2.0 ** -16 + 2.0 ** -24 * want
    assert bool(((out.logprob.cpu().double() + want).abs() <= tol).all())
    assert bool(((out.entropy.cpu().double() - want).abs() <= tol).all())
    first = [sorted(at[:int(k)])[:2] for k in n]
    assert out.top_tokens.tolist() == first
    assert out.rank.tolist() == [sorted(at[:int(k)]).index(at[1]) for k in n]
    assert not math.isnan(float(out.top_logprobs.sum()))
