"""GPU tests of polarengine_vllm.kernels.logprobs against float64 on the CPU.

Tolerances. Ranks and tokens are whole numbers and have to be equal. With exponents
relative to the row's maximum an exponential of fp32 is off by its argument's rounding,
2^-24 |x - max| <= 2^-17 for what counts (below e^-104 nothing does), and a few units of
2^-24; sums are off by less than their terms are, relative. So log sum exp is off by
less than 2^-16, the differences x - max by 2^-24 of themselves, and a log probability by
2^-16 and half a step of the result; the entropy, a mean of values of at most lse + 104,
by 2^-16 (1 + H) and half a step."""

import math

import numpy as np
import pytest
import torch

from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu


def _lp():
    from polarengine_vllm.kernels import logprobs
    return logprobs


def _check(logits, tokens, top):
    out = _lp().token_logprobs(logits, tokens, top)
    x, tok = logits.cpu().double(), tokens.cpu()
    vocab = x.shape[1]
    m = x.amax(-1, keepdim=True)
    lse = m[:, 0] + (x - m).exp().sum(-1).log()
    lp = x - lse[:, None]
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    there = (tok >= 0) & (tok < vocab)
    at = tok.clamp(0, vocab - 1)[:, None]
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    rank = torch.where(there, (order == at).int().argmax(-1), -1)
    assert torch.equal(out.rank.cpu(), rank)
    ids = order[:, :top]
    assert torch.equal(out.top_tokens.cpu(), ids)
    eps = 2.0 ** -24

    def near(got, want, tol):
        got = got.cpu().double()
        assert torch.equal(got.isinf(), want.isinf()) and not got.isnan().any()
        off = ((got - want).abs() / (tol + eps * want.abs())).nan_to_num(0.0)
        assert off.numel() == 0 or off.max() <= 1, f"error {off.max():.3f} of the tolerance"

    want = torch.where(there, lp.gather(1, at)[:, 0], 0.0)
    far = torch.where(want.isinf(), 0.0, want.abs())
    near(out.logprob, want, 2.0 ** -16 + 2 * eps * far)
    near(out.top_logprobs, lp.gather(1, ids), 2.0 ** -16 + 2 * eps * lp.gather(1, ids).abs().nan_to_num(posinf=0.0))
    near(out.entropy, entropy, 2.0 ** -16 * (1 + entropy))
    return out


def _logits(g, rows, vocab, kind):
    x = torch.randn(rows, vocab, generator=g) * 2
    if kind == "likely":
        at = torch.randint(0, vocab, (rows, 4), generator=g)
        x.scatter_(1, at, 20 + 5 * torch.rand(rows, 4, generator=g))
    if kind == "filtered":
        least = x.topk(min(7, vocab), -1).values[:, -1:]
        x = x.masked_fill(x < least, -math.inf)
    if kind == "ties":
        x = x.round()
    if kind == "same":
        x = torch.zeros(rows, vocab)
        x[:, ::3] = -0.0
    if kind == "far":
        x = x * 500 - 3000
    return x


@pytest.mark.parametrize("kind", ["random", "likely", "filtered", "ties", "same", "far"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 100, 1000, 4099, 33333])
def test_logprobs(kind, dtype, vocab):
    say(f"logprobs {kind} {dtype} vocab={vocab}")
    g = torch.Generator().manual_seed(vocab)
    for rows, top in ((1, 20), (5, 0), (9, 1), (3, 64)):
        top = min(top, vocab)
        x = _logits(g, rows, vocab, kind).to(dtype).to(DEV)
        tokens = torch.randint(0, vocab, (rows,), generator=g)
        tokens[rows // 2] = [-1, vocab, 1 << 40, -(1 << 40), 0][rows % 5]
        if rows > 4:
            tokens[0], tokens[1] = x[0].cpu().float().argmax(), vocab - 1
        _check(x, tokens.to(DEV), top)


@pytest.mark.parametrize("rows", [1, 2, 7, 40, 300])
def test_rows_of_a_large_vocabulary(rows):
    say(f"logprobs rows={rows} of 151936")
    g = torch.Generator().manual_seed(rows)
    for dtype, top in ((torch.float32, 20), (torch.bfloat16, 5)):
        x = _logits(g, min(rows, 40), 151936, "likely").to(dtype).to(DEV)
        x = x.repeat(-(-rows // x.shape[0]), 1)[:rows]
        tokens = torch.randint(0, 151936, (rows,), generator=g).to(DEV)
        if rows <= 40:
            _check(x, tokens, top)
        else:  # repeated rows repeat their answers, whatever the number of rows
            got = _lp().token_logprobs(x, tokens, top)
            part = _lp().token_logprobs(x[:40], tokens[:40], top)
            assert torch.equal(got.top_tokens[40:80], part.top_tokens)
            assert torch.equal(got.top_tokens[:40], part.top_tokens)
            assert torch.equal(got.rank[:40], part.rank)
            _check(x[260:300], tokens[260:300], top)


def test_rising_and_falling_rows():
    """Every value is larger, or smaller, than all before it."""
    for vocab in (5000, 40001):
        up = torch.arange(vocab, dtype=torch.float32) / 64
        x = torch.stack([up, up.flip(0), torch.cat([up[vocab // 2:], up[:vocab // 2]])]).to(DEV)
        _check(x, torch.tensor([0, 5, vocab - 1], device=DEV), 64)


def test_strided_rows():
    say("logprobs strided rows")
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(6, 1003, generator=g).to(DEV)
    tokens = torch.tensor([0, 5, 999, 7, 8, 9], device=DEV)
    _check(wide[:, 1:1001], tokens, 5)
    _check(wide[:, :1000].bfloat16()[:, 3:], tokens.clamp(max=996), 5)
    _check(wide[::2], tokens[:3], 5)
    _check(wide[:1000].t()[:500, :].contiguous().t()[:, :400], tokens.clamp(max=399), 3)
    _check(torch.randn(7, 6, generator=g).to(DEV).t(), tokens.clamp(max=6), 3)


def test_rows_without_a_distribution():
    """NaN, +inf and rows of -inf answer something, and leave the other rows alone."""
    say("logprobs rows without a distribution")
    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 5000, generator=g).to(DEV)
    tokens = torch.arange(6, device=DEV)
    want = _lp().token_logprobs(x, tokens, 8)
    x[1, 77], x[3] = float("nan"), -math.inf
    x[5, 3::7] = float("nan")  # ruled out
    ruled = x.clone()
    ruled[5, 3::7] = -math.inf
    want = [torch.cat([w[:5], o[5:]]) for w, o in zip(want, _lp().token_logprobs(ruled, tokens, 8))]
    x[4, 4000] = math.inf
    got = _lp().token_logprobs(x, tokens, 8)
    for w, o in zip(want, got):
        assert torch.equal(w[[0, 2, 5]], o[[0, 2, 5]])
    assert (got.top_tokens >= -1).all() and (got.top_tokens < 5000).all()


def test_captured_and_two_at_once():
    lp = _lp()
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(3, 50000, generator=g, device=DEV)
    tokens = torch.tensor([1, 2, 3], device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lp.token_logprobs(x, tokens, 10)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = lp.token_logprobs(x, tokens, 10)
    torch.cuda.synchronize()
    for i in range(6):
        x.copy_(torch.randn(3, 50000, generator=g, device=DEV) * (i + 1))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        other = torch.randn(3, 50000, generator=g, device=DEV)
        lp.token_logprobs(other, tokens, 10)
        torch.cuda.synchronize()
        for a, b in zip(out, lp.token_logprobs(x, tokens, 10)):
            assert torch.equal(a, b)


def test_gradients_are_refused():
    x = torch.randn(2, 10, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        _lp().token_logprobs(x, torch.tensor([1, 2], device=DEV))
    with torch.no_grad():
        _lp().token_logprobs(x, torch.tensor([1, 2], device=DEV))
