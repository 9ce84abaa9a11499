"""GPU tests of DecodeRunner over a paged 8-bit cache: every write and every attention
of its steps against the statements and tolerances of the operators' own tests, steps
replayed from a graph, and scores against the logits of the same step."""

import math

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_paged_cache import _attend_check, _attend_ref, _i64, _top, _write_ref
from test_gpu_tree_runner import _runner, _tokens

pytestmark = pytest.mark.gpu


def _pc():
    from polarengine_vllm.kernels import paged_cache
    return paged_cache


@pytest.mark.parametrize("qk_norm", [False, True])
def test_every_stage_of_the_steps(qk_norm, monkeypatch):
    pc = _pc()
    run = _runner(1, 200, qk_norm=qk_norm)
    pool = run.paged_pool(blocks=20, batch=4, block_size=16)
    made = []

    def write(k, v, cache, slots):
        before = pc.PagedCache(*(x.cpu() for x in cache))
        real_write(k, v, cache, slots)
        for codes, scale, x, by_dim, got in [(before.k, before.k_scale, k, False, (cache.k, cache.k_scale)),
                                             (before.v, before.v_scale, v, True, (cache.v, cache.v_scale))]:
            want = codes.float().double().numpy()
            exps = scale.view(torch.uint8).numpy().astype(int) - 127
            _write_ref(want, exps, x.cpu().double().numpy(), slots.tolist(), 16, by_dim)
            assert (got[0].cpu().float().double().numpy() == want).all()
            assert (got[1].view(torch.uint8).cpu().numpy().astype(int) - 127 == exps).all()
        made.append("write")

    def attention(q, cache, tables, starts, lengths, window, sinks):
        got = real_attention(q, cache, tables, starts, lengths, window, sinks)
        host = pc.PagedCache(*(x.cpu() for x in cache))
        out, mag = _attend_ref(q.cpu(), host, tables.tolist(), starts.tolist(), lengths.tolist(), window, sinks,
                               1 / math.sqrt(q.shape[2]))
        _attend_check(got, out, mag, q.dtype, _top(host))
        made.append("attention")
        return got

    real_write, real_attention = pc.write_blocks, pc.paged_attention
    monkeypatch.setattr(pc, "write_blocks", write)
    monkeypatch.setattr(pc, "paged_attention", attention)
    pool.keep(_i64([0, 0, -1, 0]).to(DEV))
    lengths = [0, 0, -1, 0]
    for step, counts in enumerate([[30, 1, 5, 0], [1, 1, 0, 17], [1, 20, 0, 1], [1, 1, 9, 1]]):
        say(f"paged runner qk_norm={qk_norm} step {step} counts {counts}")
        logits = run.paged_step(_tokens((40,), step), _i64(counts).to(DEV), pool, window=24, sinks=3)
        assert logits.shape == (4, 300) and bool(torch.isfinite(logits).all())
        lengths = [n + c if n >= 0 else n for n, c in zip(lengths, counts)]
        assert pool.lengths.tolist() == lengths
    assert made == ["write", "attention"] * 8
    # one is done, another takes its place; the last two tokens of a third are taken back
    pool.keep(_i64([0, lengths[1] - 2, -1, 1 << 40]).to(DEV))
    assert pool.lengths.tolist() == [0, lengths[1] - 2, -1, lengths[3]]
    run.paged_step(_tokens((40,), 9), _i64([40, 0, 0, 0]).to(DEV), pool)
    assert pool.lengths.tolist() == [40, lengths[1] - 2, -1, lengths[3]]


def test_chunks_and_layouts_of_a_step():
    """What a sequence's step writes and answers does not depend on who else is in the
    step, on which blocks it has, or on rows behind the last sequence's. Steps of 80 rows
    each, so that the linears' kernels are the same and codes have to be equal (a
    rounding of bf16, 2^-9, may move a code next to a border by its step, 2^-3 of it, so
    behind an attention whose sums are cut elsewhere they need not be: one layer); the
    logits behind the attention are roundings of bf16 apart."""
    tokens = _tokens((50,), 1)
    got = []
    for order in range(3):
        run = _runner(1, 128, layers=1)
        pool = run.paged_pool(blocks=40, batch=3, block_size=32)
        pool.keep(_i64([0, 0, 0]).to(DEV))
        say(f"paged step, arrangement {order}")
        if order == 2:
            run.paged_step(_tokens((80,), 4), _i64([33, 0, 0]).to(DEV), pool)
        head = _tokens(([0, 7, 1][order],), 2)
        step = torch.cat([head, tokens, _tokens((30 - len(head),), 3)])
        counts = [[50, 0, 0], [7, 50, 4], [1, 0, 50]][order]
        logits = run.paged_step(step, _i64(counts).to(DEV), pool)[order]
        ids = pool.tables[order, :2].long()
        cache = pool.caches[0]
        got.append((logits, cache.k.view(torch.uint8)[ids].transpose(1, 2).flatten(0, 1)[:50],
                    cache.v.view(torch.uint8)[ids].permute(0, 3, 1, 2).flatten(0, 1)[:50],
                    cache.k_scale.view(torch.uint8)[ids], cache.v_scale.view(torch.uint8)[ids]))
    for other in got[1:]:
        for a, b in zip(other[1:], got[0][1:]):
            assert torch.equal(a, b)
        err = float((other[0] - got[0][0]).abs().max() / got[0][0].abs().max())
        assert err <= 3e-2, err


def test_scores_are_those_of_the_logits():
    say("paged runner scores")
    from polarengine_vllm.kernels.logprobs import token_logprobs
    run, same = _runner(1, 128), _runner(1, 128)
    pools = [r.paged_pool(blocks=30, batch=3, block_size=16) for r in (run, same)]
    tokens, counts = _tokens((45,), 5), _i64([20, 0, 17]).to(DEV)
    for p in pools:
        p.keep(_i64([0, 0, 0]).to(DEV))
    out = run.score(tokens, counts, pools[0], top=4)
    _, attend = same._paged(tokens, counts, pools[1], None, 0)
    logits = same._layers(tokens, attend)
    follow = torch.full((45,), -1, device=DEV)
    follow[:19], follow[20:36] = tokens[1:20], tokens[21:37]
    for got, want in zip(out, token_logprobs(logits, follow, 4)):
        assert torch.equal(got, want)
    assert out.rank[19] == -1 and out.rank[36] == -1 and bool((out.logprob[:19] < 0).all())


def test_captured_steps():
    """Greedy decoding of several sequences, replayed, against the same steps run eagerly;
    a prompt joins in between."""
    run, same = _runner(1, 128), _runner(1, 128)
    pools = [r.paged_pool(blocks=30, batch=3, block_size=16) for r in (run, same)]
    prompt = _tokens((24,), 6)
    for r, p in zip((run, same), pools):
        p.keep(_i64([0, 0, -1]).to(DEV))
        r.paged_step(prompt, _i64([10, 14, 0]).to(DEV), p)
    tokens, counts = torch.zeros(3, dtype=torch.int64, device=DEV), _i64([1, 1, 0]).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        scratch = run.paged_pool(blocks=30, batch=3, block_size=16)
        run.paged_step(tokens, counts, scratch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            logits = run.paged_step(tokens, counts, pools[0])
    torch.cuda.synchronize()
    for i in range(20):
        say(f"paged replay {i}")
        graph.replay()
        want = same.paged_step(tokens, counts, pools[1])
        torch.cuda.synchronize()
        live = pools[1].lengths >= 0
        assert torch.equal(logits[:2], want[:2]) and torch.equal(pools[0].lengths, pools[1].lengths)
        tokens[:2] = logits[:2].argmax(-1)
        if i == 9:  # a third sequence
            for r, p in zip((run, same), pools):
                p.keep(torch.where(live, p.lengths, 0))
                r.paged_step(prompt[:5], _i64([0, 0, 5]).to(DEV), p)
            counts.copy_(_i64([1, 1, 1]))


def test_steps_without_room():
    """A pool that is too small: the sequence's length stays, and others go on."""
    say("paged runner without room")
    run = _runner(1, 64)
    pool = run.paged_pool(blocks=3, batch=2, block_size=16)
    pool.keep(_i64([0, 0]).to(DEV))
    run.paged_step(_tokens((40,), 7), _i64([32, 8]).to(DEV), pool)
    assert pool.lengths.tolist() == [32, 8] and pool.free_count.item() == 0
    run.paged_step(_tokens((2,), 8), _i64([1, 1]).to(DEV), pool)
    assert pool.lengths.tolist() == [32, 9]
    pool.keep(_i64([-1, 9]).to(DEV))
    assert pool.lengths.tolist() == [-1, 9] and pool.free_count.item() == 2
    for _ in range(3):
        run.paged_step(_tokens((20,), 8), _i64([5, 20]).to(DEV), pool)
    assert pool.lengths.tolist() == [-1, 29]


def test_refusals():
    run = _runner(1, 64)
    pool = run.paged_pool(blocks=3, batch=2, block_size=16)
    counts = _i64([1, 1]).to(DEV)
    with pytest.raises(ValueError):
        run.paged_step(_tokens((2, 1), 0), counts, pool)
    with pytest.raises(ValueError):
        run.paged_step(_tokens((2,), 0).int(), counts, pool)
    with pytest.raises(ValueError):
        run.paged_step(_tokens((0,), 0), counts, pool)
    with pytest.raises(ValueError):
        _runner(1, 32).paged_step(_tokens((2,), 0), counts, pool)
    with pytest.raises(ValueError):
        _runner(1, 64, layers=1).paged_step(_tokens((2,), 0), counts, pool)
    with pytest.raises(ValueError):
        run.paged_pool(blocks=3, batch=0, block_size=16)
    with pytest.raises(ValueError):
        run.paged_pool(blocks=3, batch=2, block_size=128)
