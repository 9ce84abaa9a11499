"""GPU tests of the drafted-token entry points: layouts at the edges of what their
documentation allows."""

import pytest
import torch

import test_gpu_tree_decode as base
from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("layers", [None, 1])
def test_keep_strides_along_one_element_are_not_looked_at(layout, layers):
    """One sequence, one head, one layer: what their strides are is of no meaning."""
    say(f"keep strides along one element {layout} {layers}")
    g = torch.Generator().manual_seed(1)
    k, v = (base._cache(1, 1, 24, 64, torch.bfloat16, y, 0.0, g, layers) for y in (layout, "row"))
    lengths, path, count = (base._i64(x).to(DEV) for x in ([5], [[0, 2, 5, 7, -1, -1, -1, -1]], [4]))
    want = [t.clone() for t in (k, v)]
    for w in want:
        w[..., 5:9, :] = w[..., [5, 7, 10, 12], :]
    lead = (3, 5) if layers is None else (3, 5, 7)
    odd = [t.as_strided(t.shape, lead + t.stride()[-2:]) for t in (k, v)]
    base._td().keep_accepted(*odd, lengths, path, count)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("layout", ["row", "col", "narrow"])
def test_caches_of_one_position(layout):
    """One place per sequence: the first token, keys by dimension too (``narrow``: the
    first place of a longer cache)."""
    say(f"caches of one position {layout}")
    td, g = base._td(), torch.Generator().manual_seed(2)
    b, heads, kv, dim = 3, 4, 2, 64
    full = 9 if layout == "narrow" else 1
    k, v = (base._cache(b, kv, full, dim, torch.bfloat16, y, 0.0)[:, :, :1]
            for y in ("row" if layout == "row" else "col", "row"))
    qkv = torch.randn(b, (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).to(DEV)
    table = torch.rand(4, dim, generator=g).to(DEV)
    lengths = base._i64([0, 1, 0]).to(DEV)  # the second has no room
    plan = td.tree_plan(base._i64([-1]).to(DEV), lengths)
    q = td.qk_norm_rope_write(qkv, heads, kv, table, plan.positions, k, v, lengths)
    _, keys = td.qk_norm_rope(qkv, heads, kv, table, plan.positions)
    vals = qkv.view(b, -1, dim)[:, heads + kv:]
    for s in (0, 2):
        assert torch.equal(k[s, :, 0], keys[s]) and torch.equal(v[s, :, 0], vals[s])
    assert float(k[1].abs().max()) == 0
    out = td.tree_attention(q.view(b, 1, heads, dim), k, v, lengths, plan.masks)
    for s in (0, 2):  # one key: its value
        assert torch.equal(out[s, 0], vals[s].repeat_interleave(2, 0))
    assert float(out[1].abs().max()) == 0
    before = k.clone(), v.clone()
    td.keep_accepted(k, v, lengths, torch.zeros(b, 1, dtype=torch.int64, device=DEV),
                     torch.ones(b, dtype=torch.int64, device=DEV))
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def test_runner_of_one_position():
    """DecodeRunner with a cache of one position."""
    say("runner of one position")
    from test_gpu_tree_runner import _runner, _tokens
    run = _runner(2, 1)
    lengths = torch.zeros(2, dtype=torch.int64, device=DEV)
    out, _, count = run.speculative_round(_tokens((2, 1)), lengths, torch.rand(2, 1, device=DEV))
    assert count.tolist() == [1, 1] and lengths.tolist() == [1, 1] and bool((out >= 0).all())


def test_runner_with_strided_tokens():
    """DecodeRunner: tokens that are no rows of memory."""
    say("runner strided tokens")
    from test_gpu_tree_runner import _runner, _tokens
    tokens, u = _tokens((2, 5)), torch.rand(2, 5, device=DEV)
    wide = _tokens((2, 11), 1)
    wide[:, ::2][:, :5] = tokens
    go = lambda t: _runner(2, 20).speculative_round(t, torch.zeros(2, dtype=torch.int64, device=DEV), u)
    want = go(tokens)
    for other in (tokens.t().contiguous().t(), wide[:, ::2][:, :5]):
        assert all(torch.equal(x, y) for x, y in zip(go(other), want))
    shared = tokens[:1].expand(2, -1)
    assert torch.equal(_runner(2, 20).tree_step(shared, torch.zeros(2, dtype=torch.int64, device=DEV)),
                       _runner(2, 20).tree_step(shared.contiguous(),
                                                torch.zeros(2, dtype=torch.int64, device=DEV)))
