"""GPU tests of the drafted-token kernels: every form of the attention with drafted
values that are not finite, and a whole step whose attention is held to the same
tolerance as an attention alone."""

import random

import pytest
import torch

import test_gpu_tree_decode as base
from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu


def _branches(n):
    """Two branches, from nodes 1 and 2."""
    return [-1, 0, 0][:n] + [1 + i % 2 for i in range(n - 3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,heads,lens", [  # rows of a KV head: every form of the kernel
    (4, 1, [70, 0]), (12, 2, [61, 130]), (24, 2, [3, 64]), (64, 4, [100, 5]),
    # sequences that several workgroups share, the last tile in a run of its own or not
    (5, 2, [4000]), (48, 1, [2500, 3000]), (64, 4, [3001])])
def test_drafted_values_that_are_not_finite(dtype, layout, dim, n, heads, lens):
    say(f"not finite {dtype} {layout} dim={dim} n={n} heads={heads} lens={lens}")
    q, k, v, lengths, masks = base._attention_case(n + dim, lens, n, heads, 1, dim, dtype, layout,
                                                   trees=[_branches(n)] * len(lens), cap=max(lens) + n + 3)
    want = base._attend_ref(q, k, v, lengths, masks, dim ** -0.5)
    rows = [i for i in range(n) if not int(masks[0, i]) >> 1 & 1]  # do not see node 1
    for bad in (float("nan"), float("inf")):
        v2 = v.clone()
        for s, length in enumerate(lens):
            v2[s, 0, length + 1, s::2] = bad
        got = base._attend(q, k, v2, lengths, masks, layout)
        base._check_attention(got[:, rows], [t[:, rows] for t in want], f"{bad}")
        for s in range(len(lens)):  # node 1 has it, where it is, and is as ever elsewhere
            seen = got[s, 1, :, s::2].float()
            assert bool((torch.isnan(seen) if bad != bad else seen == bad).all())
            rest = [i for i in range(dim) if i < s or (i - s) % 2]
            base._check_attention(got[s, 1][:, rest], [t[s, 1][:, rest] for t in want], "node 1")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("seed,lens,n", [(3, [30, 0, 64], 11), (4, [700, 3], 33), (5, [1500], 2)])
def test_round_by_stages(dtype, layout, seed, lens, n):
    """A step as it is used: every stage against float64, from the very tensors that the
    stage before it left."""
    say(f"round by stages {dtype} {layout} {lens} n={n}")
    td, b = base._td(), len(lens)
    s = base._round_state(seed, lens, n, layout, dtype)
    g = torch.Generator().manual_seed(seed)
    for name in ("k", "v"):  # what earlier steps left
        s[name].copy_(torch.randn(s[name].shape, generator=g).to(dtype))
    plan = td.tree_plan(s["parents"], s["lengths"])
    masks = [base._bits(t) for t in s["parents"].tolist()]
    pos = base._i64([[length + bin(m).count("1") - 1 for m in ms] for length, ms in zip(lens, masks)])
    signed = base._i64([[base._signed(m) for m in ms] for ms in masks])
    assert plan.positions.tolist() == pos.tolist() and plan.masks.tolist() == signed.tolist()
    w, scale = s["w"].cpu(), 128 ** -0.5
    for i, qkv in enumerate(s["qkv"]):
        before = [s[name][i].cpu().clone() for name in ("k", "v")]
        q = td.qk_norm_rope_write(qkv, 4, 2, s["table"], plan.positions, s["k"][i], s["v"][i],
                                  s["lengths"], s["w"], s["w"], base.EPS)
        (q_ref, q_size), (k_ref, k_size) = base._rope_ref(qkv.cpu(), 4, 2, s["table"].cpu(), pos.view(-1),
                                                          w, w)
        base._close16(q, q_ref, q_size, f"queries {i}")
        after = [s[name][i].cpu() for name in ("k", "v")]
        rows = qkv.cpu().view(b, n, 8, 128)
        for j, length in enumerate(lens):
            new = slice(length, length + n)
            base._close16(after[0][j, :, new].transpose(0, 1), k_ref.view(b, n, 2, 128)[j],
                          k_size.view(b, n, 2, 128)[j], f"keys {i}")
            assert torch.equal(after[1][j, :, new].transpose(0, 1), rows[j, :, 6:])
            for old, have in zip(before, after):  # the others are as they were
                rest = torch.ones(old.shape[2], dtype=torch.bool)
                rest[new] = False
                assert torch.equal(old[j][:, rest], have[j][:, rest])
        out = td.tree_attention(q.view(b, n, 4, 128), s["k"][i], s["v"][i], s["lengths"], plan.masks)
        want = base._attend_ref(q.cpu().view(b, n, 4, 128), *after, base._i64(lens), signed, scale)
        base._check_attention(out, want, f"layer {i}")
    got = td.verify_drafts(s["logits"], s["tokens"], s["u"], parents=s["parents"])
    want = base._verify_ref(s["logits"].cpu(), s["tokens"].cpu(), s["u"].cpu(), s["parents"].cpu(), None,
                            torch.ones(b))
    for x, y in zip(got, want):
        assert x.tolist() == y.tolist()
    kept = [s[name].cpu().clone() for name in ("k", "v")]
    td.keep_accepted(s["k"], s["v"], s["lengths"], got[1], got[2])
    for t, name in zip(kept, ("k", "v")):
        for j, length in enumerate(lens):
            src = [length + p for p in got[1][j].tolist() if p >= 0]
            t[:, j, :, length:length + len(src)] = t[:, j][:, :, src].clone()
        assert torch.equal(s[name].cpu(), t), name
