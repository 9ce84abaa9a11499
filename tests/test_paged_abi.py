"""CPU tests of the paged cache's and the log probabilities' entry points: argument
checks of the C ABI (every call below is refused, or has nothing to do, before anything
is launched: pointers are aligned placeholders) and of the Python functions."""

import pytest
import torch

OK, NULL, DIMS, ALIGN, DTYPE, WORKSPACE = 0, 1, 2, 4, 5, 6
F16, BF16, F32 = 0, 1, 2
P = 4096  # a placeholder


def _lib():
    from polarengine_vllm import _lib
    return _lib.lib()


def _change(args, **new):
    assert not new.keys() - args.keys()
    return [new.get(k, v) for k, v in args.items()]


def test_plan_step():
    a = dict(lengths=P, counts=P, tables=P, t_b=9, batch=3, width=9, free=P, cap=50, count=P, rows=7,
             block=16, starts=P, pos=P, slots=P, out=P, st=None)
    f = _lib().pe_plan_step
    assert f(*_change(a, batch=0)) == OK
    assert f(*_change(a, batch=0, rows=0, pos=None, slots=None)) == OK
    for new, rc in [({k: None}, NULL) for k in ("lengths", "counts", "tables", "free", "count", "starts",
                                                "pos", "slots", "out")] + [
            (dict(block=8), DIMS), (dict(block=48), DIMS), (dict(block=256), DIMS), (dict(batch=-1), DIMS),
            (dict(batch=4097), DIMS), (dict(width=0), DIMS), (dict(width=1 << 25, t_b=1 << 25), DIMS),
            (dict(t_b=8), DIMS), (dict(cap=0), DIMS), (dict(cap=1 << 31), DIMS), (dict(rows=-1), DIMS),
            (dict(rows=(1 << 24) + 1), DIMS)]:
        assert f(*_change(a, **new)) == rc, new


def test_release_blocks():
    a = dict(tables=P, t_b=9, batch=3, width=9, keep=P, free=P, cap=50, count=P, block=16, st=None)
    f = _lib().pe_release_blocks
    assert f(*_change(a, batch=0)) == OK
    for new, rc in [({k: None}, NULL) for k in ("tables", "keep", "free", "count")] + [
            (dict(block=0), DIMS), (dict(batch=4097), DIMS), (dict(width=0), DIMS), (dict(t_b=8), DIMS),
            (dict(cap=0), DIMS)]:
        assert f(*_change(a, **new)) == rc, new


CACHE = dict(kc=P, k_b=16384, vc=P, v_b=16384, ks=P, vs=P, s_b=2, blocks=5, kvh=2, block=64, dim=128)
CACHE_BAD = [({k: None}, NULL) for k in ("kc", "vc", "ks", "vs")] + [
    (dict(k_b=16368), DIMS), (dict(v_b=16368), DIMS), (dict(s_b=1), DIMS), (dict(blocks=0), DIMS),
    (dict(blocks=1 << 31), DIMS), (dict(kvh=0), DIMS), (dict(kvh=4097), DIMS), (dict(block=40), DIMS),
    (dict(dim=96), DIMS), (dict(dim=512), DIMS), (dict(kc=P + 8), ALIGN), (dict(vc=P + 8), ALIGN),
    (dict(k_b=16392), ALIGN), (dict(v_b=16392), ALIGN), (dict(k_b=1 << 31), DIMS), (dict(v_b=1 << 31), DIMS),
    (dict(s_b=1 << 31), DIMS)]


def test_write_blocks():
    a = dict(k=P, v=P, dtype=BF16, rows=4, k_r=768, k_h=128, v_r=768, v_h=128, slots=P)
    cache = {k: CACHE[k] for k in ("kc", "k_b", "vc", "v_b", "ks", "vs", "s_b", "blocks", "kvh", "block",
                                   "dim")}
    a.update(cache, st=None)
    f = _lib().pe_write_blocks
    assert f(*_change(a, rows=0)) == OK
    for new, rc in CACHE_BAD + [
            (dict(k=None), NULL), (dict(v=None), NULL), (dict(slots=None), NULL), (dict(dtype=F32), DTYPE),
            (dict(dtype=9), DTYPE), (dict(rows=-1), DIMS), (dict(rows=(1 << 24) + 1), DIMS),
            (dict(k_r=-8), DIMS), (dict(v_h=-8), DIMS), (dict(k=P + 2), ALIGN), (dict(v=P + 8), ALIGN),
            (dict(k_r=772), ALIGN), (dict(v_h=132), ALIGN)]:
        assert f(*_change(a, **new)) == rc, new


def test_paged_attention():
    a = dict(q=P, dtype=BF16, q_r=1024, rows=4, heads=8)
    a.update(CACHE, tables=P, t_b=9, batch=3, width=9, starts=P, lengths=P, window=0, sinks=0, scale=0.1,
             out=P, ws=P, ws_bytes=1 << 30, st=None)
    L = _lib()
    f = L.pe_paged_attention
    assert f(*_change(a, rows=0)) == OK
    for new, rc in CACHE_BAD + [({k: None}, NULL) for k in ("q", "tables", "starts", "lengths", "out")] + [
            (dict(dtype=F32), DTYPE), (dict(rows=-1), DIMS), (dict(batch=4097), DIMS), (dict(batch=-1), DIMS),
            (dict(width=0), DIMS), (dict(t_b=8), DIMS), (dict(heads=0), DIMS), (dict(heads=7), DIMS),
            (dict(heads=65536), DIMS), (dict(q_r=-8), DIMS), (dict(window=-1), DIMS), (dict(sinks=-1), DIMS),
            (dict(scale=float("nan")), DIMS), (dict(scale=-1.0), DIMS), (dict(scale=float("inf")), DIMS),
            (dict(q=P + 2), ALIGN), (dict(q_r=1028), ALIGN), (dict(out=P + 8), ALIGN)]:
        assert f(*_change(a, **new)) == rc, new
    need = L.pe_paged_attention_workspace_size(4, 3, 8, 2, 128, 9 * 64)
    if need:
        assert f(*_change(a, ws=None)) == WORKSPACE
        assert f(*_change(a, ws_bytes=need - 1)) == WORKSPACE
        assert f(*_change(a, ws=P + 4)) == ALIGN


def test_token_logprobs():
    a = dict(logits=P, dtype=F32, rows=3, ld=1000, vocab=1000, tokens=P, top=5, lp=P, rank=P, ent=P, tl=P,
             tt=P, ws=P, ws_bytes=1 << 30, st=None)
    L = _lib()
    f = L.pe_token_logprobs
    assert f(*_change(a, rows=0)) == OK
    for new, rc in [({k: None}, NULL) for k in ("logits", "tokens", "lp", "rank", "ent", "tl", "tt")] + [
            (dict(dtype=3), DTYPE), (dict(rows=-1), DIMS), (dict(rows=1 << 24), DIMS), (dict(logits=P + 2), ALIGN),
            (dict(vocab=0), DIMS), (dict(ld=999), DIMS),
            (dict(vocab=(1 << 24) + 1, ld=1 << 25), DIMS), (dict(top=-1), DIMS), (dict(top=65), DIMS),
            (dict(top=5, vocab=4), DIMS)]:
        assert f(*_change(a, **new)) == rc, new
    need = L.pe_token_logprobs_workspace_size(3, 1000, 5)
    if need:
        assert f(*_change(a, ws=None)) == WORKSPACE
        assert f(*_change(a, ws_bytes=need - 1)) == WORKSPACE


# ---------------------------------------------------------------------------
# Python checks: what is refused before a device is asked for is refused on the CPU
# ---------------------------------------------------------------------------
def _cpu_as_gpu(monkeypatch, module):
    """The module's functions with CPU tensors; calls into the library are counted."""
    made = []
    monkeypatch.setattr(module, "inputs", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(module, "call", lambda name, dev, *a: made.append(name))
    return made


def test_python_cache_checks(monkeypatch):
    from polarengine_vllm.kernels import paged_cache as pc
    made = _cpu_as_gpu(monkeypatch, pc)
    cache = pc.new_cache(6, 2, 16, 64, "cpu")
    assert cache.k.shape == (6, 2, 16, 64) and cache.v.shape == (6, 2, 64, 16)
    with pytest.raises(ValueError):
        pc.new_cache(6, 2, 24, 64, "cpu")
    with pytest.raises(ValueError):
        pc.new_cache(6, 2, 16, 80, "cpu")
    with pytest.raises(ValueError):
        pc.new_cache(0, 2, 16, 64, "cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.arange(3)
    pc.write_blocks(k, k, cache, slots)
    every = pc.PagedCache(*(t[::2] for t in cache))  # strided blocks
    pc.write_blocks(k, k, every, slots)
    one = pc.PagedCache(*(t[:1] for t in cache))
    pc.write_blocks(k, k, one, slots)
    assert made == ["pe_write_blocks"] * 3
    bad = [cache._replace(k=cache.k.view(torch.uint8)), cache._replace(k_scale=cache.k_scale.view(torch.uint8)),
           cache._replace(v=cache.k), cache._replace(k=cache.k[:5]), cache._replace(v_scale=cache.v_scale[:, :1]),
           cache._replace(k=cache.v.transpose(2, 3)), cache._replace(v=cache.k.transpose(2, 3)),
           cache._replace(k=cache.k[:, :, :8]), cache._replace(k=cache.k[:1].expand(6, 2, 16, 64)),
           cache._replace(k_scale=cache.k_scale[:1].expand(6, 2)),
           cache._replace(v_scale=cache.k_scale)]
    for c in bad:
        with pytest.raises((ValueError, TypeError)):
            pc.write_blocks(k, k, c, slots)
    for args in [(k.float(), k.float(), cache, slots), (k, k.half(), cache, slots), (k, k[:2], cache, slots),
                 (k[:, :1], k[:, :1], cache, slots), (k, k, cache, slots[:2]), (k, k, cache, slots.int())]:
        with pytest.raises((ValueError, TypeError)):
            pc.write_blocks(*args)
    assert len(made) == 3


def test_python_attention_checks(monkeypatch):
    from polarengine_vllm.kernels import paged_cache as pc
    made = _cpu_as_gpu(monkeypatch, pc)
    cache = pc.new_cache(6, 2, 16, 64, "cpu")
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    tables = torch.zeros(2, 5, dtype=torch.int32)
    starts, lengths = torch.tensor([0, 1, 3]), torch.tensor([9, 20])
    good = dict(q=q, cache=cache, tables=tables, starts=starts, lengths=lengths)
    pc.paged_attention(**good)
    pc.paged_attention(**good, window=1, sinks=0, scale=0.5)
    assert made == ["pe_paged_attention"] * 2
    for new in [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q[:, :0]),
                dict(tables=tables.long()), dict(tables=tables[:1]), dict(tables=tables[:, :0]),
                dict(starts=starts[:2]), dict(starts=starts.int()), dict(lengths=lengths[None]),
                dict(lengths=lengths.int()), dict(window=0), dict(window=-4), dict(sinks=-1)]:
        with pytest.raises((ValueError, TypeError)):
            pc.paged_attention(**{**good, **new})
    assert len(made) == 2
    out = pc.paged_attention(q[:0], cache, tables, starts, lengths)
    assert out.shape == (0, 4, 64) and len(made) == 2
    out = pc.paged_attention(q, cache, tables[:0], starts[:1], lengths[:0])
    assert out.shape == q.shape and not out.any() and len(made) == 2


def test_python_plan_checks(monkeypatch):
    from polarengine_vllm.kernels import paged_cache as pc
    made = _cpu_as_gpu(monkeypatch, pc)
    two = torch.tensor([3, 4])
    tables, free, count = torch.zeros(2, 5, dtype=torch.int32), torch.zeros(9, dtype=torch.int32), torch.tensor([9])
    good = [two, two, tables, free, count, 8, 16]
    plan = pc.plan_step(*good)
    assert [t.shape[0] for t in plan] == [3, 8, 8, 2] and made == ["pe_plan_step"]
    pc.release_blocks(tables, two, free, count, 16)
    empty = pc.plan_step(two[:0], two[:0], tables[:0], free, count, 3, 16)
    assert empty.slots.tolist() == [-1] * 3 and empty.starts.tolist() == [0] and len(made) == 2
    for i, new in [(0, two.int()), (0, two[None]), (1, two[:1]), (2, tables.long()), (2, tables[:1]),
                   (2, tables.t()), (2, tables[:1].expand(2, 5)), (2, tables[:, :0]), (3, free.long()),
                   (3, free[:0]), (3, free[::2]), (4, count.int()), (4, two), (5, -1), (6, 24)]:
        args = list(good)
        args[i] = new
        with pytest.raises((ValueError, TypeError)):
            pc.plan_step(*args)
    for i, new in [(0, tables.long()), (0, tables[:, ::2]), (1, two[:1]), (1, two.int()), (2, free.long()),
                   (3, count.int()), (4, 17)]:
        args = [tables, two, free, count, 16]
        args[i] = new
        with pytest.raises((ValueError, TypeError)):
            pc.release_blocks(*args)
    assert len(made) == 2


def test_python_logprob_checks(monkeypatch):
    from polarengine_vllm.kernels import logprobs as lp
    made = _cpu_as_gpu(monkeypatch, lp)
    x, tok = torch.zeros(2, 10), torch.tensor([1, 2])
    out = lp.token_logprobs(x, tok, 3)
    assert out.top_tokens.shape == (2, 3) and out.rank.shape == (2,) and made == ["pe_token_logprobs"]
    assert lp.token_logprobs(x[:0], tok[:0]).logprob.shape == (0,)
    for args in [(x.double(), tok), (x[0], tok), (x[:, :0], tok), (x, tok[:1]), (x, tok.int()), (x, tok, -1),
                 (x, tok, 11), (torch.zeros(2, 100), tok, 65)]:
        with pytest.raises((ValueError, TypeError)):
            lp.token_logprobs(*args)
    assert len(made) == 1


def test_cpu_tensors_and_gradients_are_refused():
    from polarengine_vllm.kernels import logprobs as lp, paged_cache as pc
    cache = pc.new_cache(6, 2, 16, 64, "cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    two = torch.tensor([0, 1])
    calls = [lambda: pc.write_blocks(k, k, cache, torch.arange(3)),
             lambda: pc.paged_attention(k, cache, torch.zeros(1, 2, dtype=torch.int32), two, two[:1]),
             lambda: pc.release_blocks(torch.zeros(2, 5, dtype=torch.int32), two,
                                       torch.zeros(9, dtype=torch.int32), two[:1], 16),
             lambda: lp.token_logprobs(torch.zeros(2, 10), two)]
    for f in calls:
        with pytest.raises(RuntimeError, match="GPU only"):
            f()
