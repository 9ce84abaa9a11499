"""CPU tests of the drafted-token entry points: argument checks of the C ABI (every
call below is refused, or has nothing to do, before anything is launched: pointers
are aligned placeholders) and of the Python functions, workspace sizes."""

import pytest
import torch

OK, NULL, DIMS, ALIGN, DTYPE, WORKSPACE = 0, 1, 2, 4, 5, 6
BF16, F32 = 1, 2
P = 4096  # a placeholder


def _lib():
    from polarengine_vllm import _lib
    return _lib.lib()


def _change(args, **new):
    return [new.get(k, v) for k, v in args.items()]


def test_tree_plan():
    a = dict(parents=P, stride=0, lengths=P, batch=2, n=4, pos=P, masks=P, st=None)
    f = _lib().pe_tree_plan
    assert f(*_change(a, batch=0)) == OK
    for new, rc in [(dict(parents=None), NULL), (dict(lengths=None), NULL), (dict(masks=None), NULL),
                    (dict(n=0), DIMS), (dict(n=65), DIMS), (dict(batch=-1), DIMS),
                    (dict(stride=-1), DIMS), (dict(batch=1 << 24), DIMS)]:
        assert f(*_change(a, **new)) == rc, new


ROPE = dict(qkv=P, dtype=BF16, rows=4, ld=768, heads=4, kv=1, dim=128, rope=P, rope_rows=9, rot=128,
            pos=P, qw=None, kw=None, eps=1e-6, q=P)
ROPE_BAD = [(dict(qkv=None), NULL), (dict(rope=None), NULL), (dict(pos=None), NULL), (dict(q=None), NULL),
            (dict(dtype=F32), DTYPE), (dict(dtype=7), DTYPE), (dict(dim=96), DIMS), (dict(dim=512), DIMS),
            (dict(rot=24), DIMS), (dict(rot=0), DIMS), (dict(rot=144), DIMS), (dict(rope_rows=0), DIMS),
            (dict(heads=0), DIMS), (dict(kv=0), DIMS), (dict(heads=65537), DIMS), (dict(ld=760), DIMS),
            (dict(ld=772), ALIGN), (dict(qkv=P + 2), ALIGN), (dict(rope=P + 4), ALIGN),
            (dict(q=P + 8), ALIGN), (dict(qw=P + 8), ALIGN), (dict(kw=P + 2), ALIGN)]


def test_qk_norm_rope():
    a = dict(ROPE, k=P, st=None)
    f = _lib().pe_qk_norm_rope
    assert f(*_change(a, rows=0)) == OK
    for new, rc in ROPE_BAD + [(dict(k=None), NULL), (dict(k=P + 2), ALIGN), (dict(rows=-1), DIMS),
                               (dict(rows=1 << 31), DIMS), (dict(rows=(1 << 31) - 1), DIMS)]:
        assert f(*_change(a, **new)) == rc, new


CACHES = dict(k=P, ksb=8192, ksh=8192, ksl=128, ksd=1, v=P, vsb=8192, vsh=8192, vsl=128)
CACHES_BAD = [(dict(ksd=2), DIMS), (dict(ksb=-8), DIMS), (dict(vsl=-128), DIMS), (dict(k=P + 2), ALIGN),
              (dict(v=P + 8), ALIGN), (dict(ksl=130), ALIGN), (dict(vsl=132), ALIGN),
              (dict(ksb=8196), ALIGN), (dict(vsl=1 << 26), DIMS), (dict(ksl=1 << 26), DIMS),
              (dict(ksl=1, ksd=1 << 26), DIMS)]


def test_qk_norm_rope_write():
    a = dict(qkv=P, dtype=BF16, batch=2, n=2)
    a.update({k: v for k, v in ROPE.items() if k not in ("qkv", "dtype", "rows")})
    a.update(CACHES, lengths=P, cap=64, st=None)
    f = _lib().pe_qk_norm_rope_write
    assert f(*_change(a, batch=0)) == OK
    bad = [(new, rc) for new, rc in ROPE_BAD + CACHES_BAD]
    for new, rc in bad + [(dict(k=None), NULL), (dict(v=None), NULL), (dict(lengths=None), NULL),
                          (dict(n=0), DIMS), (dict(cap=0), DIMS), (dict(batch=-1), DIMS),
                          (dict(n=1 << 31), DIMS), (dict(batch=1 << 20, n=1 << 20), DIMS)]:
        assert f(*_change(a, **new)) == rc, new


def test_tree_attention():
    a = dict(q=P, dtype=BF16, qb=2048, qn=512, **CACHES, lengths=P, masks=P, mb=4, out=P, batch=2, n=4,
             heads=4, kvh=1, dim=128, cap=1000, scale=0.1, ws=P, ws_bytes=1 << 30, st=None)
    L = _lib()
    f = L.pe_tree_attention
    assert f(*_change(a, batch=0)) == OK
    size = L.pe_tree_attention_workspace_size
    need = size(2, 4, 4, 1, 128, 1000)
    assert need > 0 and size(2, 4, 4, 1, 128, 64) == 0  # one tile: nothing to divide
    assert size(2, 65, 4, 1, 128, 1000) == 0 and size(2, 4, 3, 2, 128, 1000) == 0
    for new, rc in CACHES_BAD + [
            (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(lengths=None), NULL),
            (dict(masks=None), NULL), (dict(out=None), NULL), (dict(dtype=F32), DTYPE),
            (dict(n=0), DIMS), (dict(n=65), DIMS), (dict(batch=65536), DIMS), (dict(heads=3, kvh=2), DIMS),
            (dict(kvh=0), DIMS), (dict(dim=96), DIMS), (dict(cap=0), DIMS), (dict(cap=1 << 31), DIMS),
            (dict(batch=65535, kvh=1024, heads=1024, cap=1 << 30), DIMS), (dict(qb=-8), DIMS),
            (dict(mb=-1), DIMS), (dict(scale=-1.0), DIMS), (dict(scale=float("nan")), DIMS),
            (dict(scale=float("inf")), DIMS), (dict(q=P + 2), ALIGN), (dict(qn=516), ALIGN),
            (dict(out=P + 8), ALIGN), (dict(ws=None), WORKSPACE), (dict(ws_bytes=need - 1), WORKSPACE),
            (dict(ws=P + 8), ALIGN)]:
        assert f(*_change(a, **new)) == rc, new


def test_verify_drafts():
    a = dict(logits=P, dtype=F32, lb=4000, ln=1000, batch=2, n=4, vocab=1000, tokens=P, parents=None,
             pb=0, u=P, temps=None, temp=1.0, probs=None, qb=0, qn=0, out=P, path=P, count=P, ws=P,
             ws_bytes=1 << 30, st=None)
    L = _lib()
    f = L.pe_verify_drafts
    assert f(*_change(a, batch=0)) == OK
    need = L.pe_verify_drafts_workspace_size(2, 4, 1000)
    assert need > 0 and L.pe_verify_drafts_workspace_size(2, 4, 0) == 0
    for new, rc in [(dict(logits=None), NULL), (dict(tokens=None), NULL), (dict(u=None), NULL),
                    (dict(out=None), NULL), (dict(path=None), NULL), (dict(count=None), NULL),
                    (dict(dtype=9), DTYPE), (dict(n=0), DIMS), (dict(n=65), DIMS), (dict(vocab=0), DIMS),
                    (dict(vocab=(1 << 24) + 1), DIMS), (dict(batch=65536), DIMS), (dict(lb=-1), DIMS),
                    (dict(parents=P, probs=P), DIMS), (dict(qb=-1), DIMS),
                    (dict(batch=65535, n=64, vocab=1 << 24), DIMS), (dict(ws=None), WORKSPACE),
                    (dict(ws_bytes=need - 1), WORKSPACE), (dict(ws=P + 4), ALIGN)]:
        assert f(*_change(a, **new)) == rc, new


def test_keep_accepted():
    a = dict(cache=P, layers=2, batch=2, heads=2, cap=64, dim=128, sl=1 << 20, sb=1 << 16, sh=8192,
             spos=128, sd=1, lengths=P, path=P, count=P, n=4, st=None)
    f = _lib().pe_keep_accepted
    assert f(*_change(a, batch=0)) == OK and f(*_change(a, layers=0)) == OK
    for new, rc in [(dict(cache=None), NULL), (dict(lengths=None), NULL), (dict(path=None), NULL),
                    (dict(count=None), NULL), (dict(n=65), DIMS), (dict(n=0), DIMS), (dict(cap=0), DIMS),
                    (dict(dim=12), DIMS), (dict(spos=2, sd=2), DIMS), (dict(layers=65536), DIMS),
                    (dict(batch=65536), DIMS), (dict(heads=0), DIMS), (dict(cache=P + 2), ALIGN),
                    (dict(spos=132), ALIGN), (dict(heads=65536, dim=4096, spos=1, sd=64), DIMS)]:
        assert f(*_change(a, **new)) == rc, new


def test_python_needs_a_gpu_and_checks_before_it_launches(monkeypatch):
    """CPU tensors are refused; past that check (replaced here) shapes, types and
    layouts are, so nothing below reaches a launch."""
    from polarengine_vllm.kernels import tree_decode as td
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    lengths, masks = torch.zeros(2, dtype=torch.int64), torch.ones(2, 3, dtype=torch.int64)
    qkv, table = torch.zeros(6, 8 * 64, dtype=torch.bfloat16), torch.zeros(16, 64)
    pos = torch.zeros(6, dtype=torch.int64)
    logits, u = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    calls = [lambda: td.tree_plan(masks, lengths), lambda: td.qk_norm_rope(qkv, 4, 2, table, pos),
             lambda: td.qk_norm_rope_write(qkv, 4, 2, table, pos, k, k.clone(), lengths),
             lambda: td.tree_attention(q, k, k, lengths, masks),
             lambda: td.verify_drafts(logits, masks, u),
             lambda: td.keep_accepted(k, k.clone(), lengths, masks, lengths)]
    for call in calls:
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    monkeypatch.setattr(td, "_inputs", lambda *t: t[0].device)

    def never(*args):
        raise AssertionError("reached a launch")

    monkeypatch.setattr(td, "_call", never)
    for err, call in [
            (ValueError, lambda: td.tree_plan(masks[:, :0], lengths)),
            (ValueError, lambda: td.tree_plan(masks[:1], lengths)),
            (TypeError, lambda: td.tree_plan(masks.int(), lengths)),
            (ValueError, lambda: td.qk_norm_rope(qkv, 4, 3, table, pos)),
            (TypeError, lambda: td.qk_norm_rope(qkv.float(), 4, 2, table, pos)),
            (TypeError, lambda: td.qk_norm_rope(qkv, 4, 2, table.half(), pos)),
            (ValueError, lambda: td.qk_norm_rope(qkv, 4, 2, table, pos[:3])),
            (ValueError, lambda: td.qk_norm_rope_write(qkv, 4, 2, table, pos, k, k, lengths)),
            (ValueError, lambda: td.qk_norm_rope_write(qkv, 4, 2, table, pos, k[:1].expand(2, -1, -1, -1),
                                                       k, lengths)),
            (ValueError, lambda: td.qk_norm_rope_write(qkv[:5], 4, 2, table, pos[:5], k, k.clone(), lengths)),
            (ValueError, lambda: td.tree_attention(q[:, :, :3], k, k, lengths, masks)),
            (TypeError, lambda: td.tree_attention(q.half(), k, k, lengths, masks)),
            (ValueError, lambda: td.tree_attention(q, k, k, lengths, masks[:, :2])),
            (ValueError, lambda: td.tree_attention(q, k, k.transpose(-1, -2).contiguous().transpose(-1, -2),
                                                   lengths, masks)),
            (ValueError, lambda: td.verify_drafts(logits, masks, u, temperature=-1.0)),
            (ValueError, lambda: td.verify_drafts(logits, masks, u, parents=masks,
                                                  draft_probs=torch.zeros(2, 2, 50))),
            (ValueError, lambda: td.verify_drafts(logits, masks[:, :2], u)),
            (TypeError, lambda: td.verify_drafts(logits.double(), masks, u)),
            (ValueError, lambda: td.keep_accepted(k[:1].expand(2, -1, -1, -1), k, lengths, masks, lengths)),
            (ValueError, lambda: td.keep_accepted(k, k.clone(), lengths, masks, lengths[:1]))]:
        with pytest.raises(err):
            call()
