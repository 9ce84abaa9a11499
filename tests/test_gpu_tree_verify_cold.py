"""GPU tests of the verification of drafted tokens at small temperatures, where
everything lies on the largest logit, against the float64 walk. Whole numbers: they
have to be equal."""

import pytest
import torch

import test_gpu_tree_decode as base
from gpu_helpers import say

pytestmark = pytest.mark.gpu

# the last is the smallest positive fp32 number
TEMPS = [1e-2, 1e-6, 1e-8, 1e-10, 1e-14, 1e-16, 1e-18, 1e-20, 1e-30, 1e-38, 1.4e-45]


def _case(seed, vocab, dtype, n=5):
    """A sequence per temperature and place of the likeliest token among the root's
    children 1 .. n - 1 (0: not drafted)."""
    b = len(TEMPS) * n
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, n, vocab, generator=g) * 5 + 20).to(dtype)
    tokens = torch.randint(0, vocab, (b, n), generator=g)
    temp = torch.tensor([TEMPS[s // n] for s in range(b)])
    u = torch.rand(b, n, generator=g)
    u[::3] = 1 - 2.0 ** -24  # the largest
    best = logits.float().argmax(-1)
    for s in range(b):
        if s % n:
            tokens[s, s % n] = best[s, 0]
    return logits, tokens, u, temp, best


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [300, 9001])
def test_siblings(dtype, vocab):
    say(f"verify cold siblings {dtype} {vocab}")
    logits, tokens, u, temp, best = _case(vocab, vocab, dtype)
    n = tokens.shape[1]
    parents = torch.tensor([-1] + [0] * (n - 1)).expand_as(tokens).contiguous()
    out, _, count = base._check_verify(logits, tokens, u, parents, None, temp)
    if dtype is torch.float32:  # no two logits alike: greedy, whatever the numbers
        assert out[:, 0].tolist() == best[:, 0].tolist()
        assert [int(c) for c in count[1:n]] == [2] * (n - 1)


@pytest.mark.parametrize("drawn", [False, True])
def test_chains(drawn):
    """Chains of each node's likeliest token: accepted whole; and, with what they were
    drawn from, chains whose third draft is not it."""
    say(f"verify cold chains drawn={drawn}")
    vocab = 777
    logits, tokens, u, temp, best = _case(5, vocab, torch.float32)
    tokens[:, 1:] = best[:, :-1]
    tokens[1::2, 3] = (tokens[1::2, 3] + 1) % vocab
    probs = None
    if drawn:
        g = torch.Generator().manual_seed(6)
        probs = torch.softmax(torch.randn(*tokens[:, 1:].shape, vocab, generator=g), -1) * 0.4
        probs.scatter_(-1, tokens[:, 1:, None], 0.6)
    _, _, count = base._check_verify(logits, tokens, u, None, probs, temp)
    # below 1e-2, where the runner-up's share is exp(-d / T) < 2^-60: the largest logits
    # of a node are d > 1e-4 apart; at 1e-2 the float64 walk alone decides
    two = logits.topk(2, -1).values
    assert float((two[..., 0] - two[..., 1]).min()) > 1e-4
    cold = [s for s in range(len(count)) if TEMPS[s // 5] < 1e-2]
    assert [int(count[s]) for s in cold] == [3 if s % 2 else 5 for s in cold]


def test_close_and_equal_logits():
    """Two largest logits alike, or one fp32 step apart, with temperatures around that
    step: both keep their share."""
    say("verify cold ties")
    b, n, vocab = 60, 3, 500
    g = torch.Generator().manual_seed(9)
    logits = torch.randn(b, n, vocab, generator=g) * 3
    top = torch.full((b, n), 23.1)
    logits[:, :, 7] = top
    logits[:, :, 401] = torch.where((torch.arange(b) % 2 == 0)[:, None], top,
                                    torch.nextafter(top, torch.zeros(())))
    tokens = torch.tensor([0, 401, 7]).expand(b, n).contiguous()
    parents = torch.tensor([-1, 0, 0]).expand(b, n).contiguous()
    temp = torch.tensor([1e-30, 1e-16, 3e-7, 1e-6, 2e-6, 1e-5])[torch.arange(b) % 6]
    base._check_verify(logits, tokens, torch.rand(b, n, generator=g), parents, None, temp)
