"""CPU tests of the drafted-token entry points: calls at the edges of what their
documentation allows. Nothing here reaches a launch: the device check and the call
into the library are replaced."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

BF = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    """The calls that would go into the library: (name, arguments)."""
    from polarengine_vllm import _lib
    from polarengine_vllm.kernels import tree_decode as td
    made = []
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(td, "_call", lambda name, dev, *args: made.append((name, args)))
    return made


def _inputs():
    q = torch.zeros(2, 3, 4, 64, dtype=BF)
    k = torch.zeros(2, 2, 16, 64, dtype=BF)
    lengths, masks = torch.zeros(2, dtype=torch.int64), torch.ones(2, 3, dtype=torch.int64)
    qkv, table = torch.zeros(6, 8 * 64, dtype=BF), torch.zeros(16, 64)
    pos = torch.zeros(6, dtype=torch.int64)
    return q, k, lengths, masks, qkv, table, pos


def test_forward_mode_tangents_are_refused(calls):
    """A dual tensor would lose its tangent; no_grad does not turn forward mode off."""
    from polarengine_vllm.kernels import tree_decode as td
    q, k, lengths, masks, qkv, table, pos = _inputs()
    logits, u = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))
        for call in (lambda: td.tree_attention(dual(q), k, k, lengths, masks),
                     lambda: td.tree_attention(q, dual(k), k, lengths, masks),
                     lambda: td.tree_attention(q, k, dual(k), lengths, masks),
                     lambda: td.qk_norm_rope(dual(qkv), 4, 2, table, pos),
                     lambda: td.qk_norm_rope(qkv, 4, 2, dual(table), pos),
                     lambda: td.qk_norm_rope(qkv, 4, 2, table, pos, dual(torch.ones(64, dtype=BF))),
                     lambda: td.qk_norm_rope_write(qkv, 4, 2, table, pos, dual(k), k.clone(), lengths),
                     lambda: td.verify_drafts(dual(logits), masks, u),
                     lambda: td.verify_drafts(logits, masks, dual(u)),
                     lambda: td.verify_drafts(logits, masks, u, temperature=dual(torch.ones(2))),
                     lambda: td.keep_accepted(dual(k), k.clone(), lengths, masks, lengths)):
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(RuntimeError, match="no backward pass"):
                    call()
        assert not calls
        td.tree_attention(q, k, k, lengths, masks)  # nothing of it is dual
    td.tree_attention(fwAD.unpack_dual(q).primal, k, k, lengths, masks)
    assert [name for name, _ in calls] == ["pe_tree_attention"] * 2


def test_strides_along_one_element(calls):
    """Along one element a stride says nothing; the one position of a cache by dimension
    keeps that layout."""
    from polarengine_vllm.kernels import tree_decode as td
    lengths, one = torch.zeros(1, dtype=torch.int64), torch.ones(1, 1, dtype=torch.int64)
    rows = torch.zeros(1, 1, 8, 64, dtype=BF).as_strided((1, 1, 8, 64), (3, 5, 64, 1))
    cols = torch.zeros(1, 1, 64, 8, dtype=BF).transpose(-1, -2).as_strided((1, 1, 8, 64), (3, 5, 1, 8))
    td.keep_accepted(cols, rows, lengths, one, lengths)
    assert [a[6:11] for _, a in calls] == [(0, 0, 0, 1, 8), (0, 0, 0, 64, 1)]
    calls.clear()
    whole = torch.zeros(2, 2, 64, 1, dtype=BF).transpose(-1, -2)
    first = torch.zeros(2, 2, 64, 9, dtype=BF).transpose(-1, -2)[:, :, :1]
    v = torch.zeros(2, 2, 1, 64, dtype=BF)
    lengths, one = torch.zeros(2, dtype=torch.int64), torch.ones(2, 1, dtype=torch.int64)
    for k, want in ((whole, (128, 64, 0, 1)), (first, (1152, 576, 1, 9))):
        td.keep_accepted(k, v, lengths, one, lengths)
        assert calls[0][1][7:11] == want and calls[1][1][7:11] == (128, 64, 0, 1)
        td.tree_attention(torch.zeros(2, 1, 4, 64, dtype=BF), k, v, lengths, one)
        assert calls[2][1][5:9] == want
        calls.clear()


@pytest.mark.parametrize("dim,per_cu", [(64, 2), (256, 1)])
@pytest.mark.parametrize("n,group", [(1, 1), (40, 8), (48, 8), (64, 10), (64, 12), (64, 40), (64, 100)])
def test_attention_runs_fit_every_xcd(dim, per_cu, n, group):
    """The row blocks of a run share an XCD of 32 CUs: no more workgroups there than they
    hold at a time (the number of runs from the workspace, two parts each)."""
    from polarengine_vllm import _lib
    rows = n * group
    block = 16 if rows <= 16 else 128
    need = _lib.lib().pe_tree_attention_workspace_size(4, n, 2 * group, 2, dim, 100000)
    blocks = -(-rows // block)
    runs, rest = divmod(need, blocks * 2 * block * (dim + 2) * 4)
    assert runs >= 1 and rest == 0
    slots = 32 * per_cu
    if blocks <= slots:
        assert -(-runs // 8) * blocks <= slots and runs * blocks > 8 * (slots - blocks)
    else:
        assert runs * blocks <= 8 * slots or runs == 1


def test_one_cache_for_keys_and_values_is_refused(calls):
    """The accepted rows of one memory would be moved twice."""
    from polarengine_vllm.kernels import tree_decode as td
    _, k, lengths, masks, qkv, table, pos = _inputs()
    for call in (lambda: td.keep_accepted(k, k, lengths, masks, lengths),
                 lambda: td.keep_accepted(k[None], k[None], lengths, masks, lengths),
                 lambda: td.qk_norm_rope_write(qkv, 4, 2, table, pos, k, k, lengths)):
        with pytest.raises(ValueError, match="same memory"):
            call()
    assert not calls
    both = torch.zeros(2, 2, 16, 128, dtype=BF)  # side by side in one tensor
    td.keep_accepted(both[..., :64], both[..., 64:], lengths, masks, lengths)
    assert len(calls) == 2


def test_nothing_moves_if_the_values_cannot(calls):
    """Values whose layout the library refuses: before the keys have moved."""
    from polarengine_vllm.kernels import tree_decode as td
    _, k, lengths, masks, *_ = _inputs()
    for v in (torch.zeros(2, 2, 16, 68, dtype=BF)[..., 4:],         # rows not 16-byte aligned
              torch.zeros(2, 2, 16, 132, dtype=BF)[..., ::2][..., :64],  # nothing contiguous
              torch.zeros(2, 2, 16, 60, dtype=BF)):
        with pytest.raises(RuntimeError, match="pe_keep_accepted"):
            td.keep_accepted(k, v, lengths, masks, lengths)
    assert not calls
