"""GPU tests of DecodeRunner's steps with several drafted tokens: against its own
one-token steps, and round after round against what verification of the step's
logits says.

The two ways through the layers round differently (bf16 residual stream, linear
outputs and attention): logits are compared as the one-token step is with its fp32
statement, normwise ||d||_inf / ||ref||_inf <= 3e-2 and cosine >= 0.999."""

import dataclasses

import pytest
import torch

from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu


def _runner(batch, max_len, seed=3, **over):
    from polarengine_vllm.decode_runner import DecodeRunner, DecoderConfig
    cfg = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, intermediate=384,
                        vocab=300)
    return DecodeRunner(dataclasses.replace(cfg, **over), batch, max_len, DEV, seed=seed)


def _near(got, want, what):
    err = float((got - want).abs().max() / want.abs().max())
    cos = float(torch.nn.functional.cosine_similarity(got.flatten(), want.flatten(), 0))
    assert err <= 3e-2 and cos >= 0.999, f"{what}: normwise {err:.3e}, cosine {cos:.6f}"


def _tokens(shape, seed=0, vocab=300):
    return torch.randint(0, vocab, shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("max_len", [48, 51])
def test_chain_step_is_the_one_token_steps(qk_norm, max_len):
    say(f"chain step qk_norm={qk_norm} max_len={max_len}")
    b, n, start = 3, 7, 5
    one, many = (_runner(b, max_len, qk_norm=qk_norm) for _ in range(2))
    tokens = _tokens((b, start + n))
    for t in range(start + n):
        pos = torch.tensor([t], device=DEV)
        want = one.step(tokens[:, t], pos)
        if t < start:
            many.step(tokens[:, t], pos)
        else:
            if t == start:
                got = many.tree_step(tokens[:, start:], torch.full((b,), start, device=DEV))
            _near(got[:, t - start], want, f"node {t - start}")
    assert bool((many.k_cache[..., start + n:] == 0).all())


def test_norms_of_queries_and_keys():
    """The one-token step with per-head norms: the kernels against torch's form."""
    say("runner qk_norm")
    b = 2
    g = torch.Generator().manual_seed(4)
    a, ref = (_runner(b, 40, qk_norm=True) for _ in range(2))
    plain = _runner(b, 40)
    for la, lr in zip(a.layers, ref.layers):
        for name in ("q_norm", "k_norm"):
            w = (1 + 0.5 * torch.randn(64, generator=g)).to(torch.bfloat16).to(DEV)
            la[name] = lr[name] = w
    ref._attention = ref._attention_torch
    for t in range(6):
        tok, pos = _tokens((b,), t), torch.tensor([t], device=DEV)
        got = a.step(tok, pos)
        _near(got, ref.step(tok, pos), f"step {t}")
        other = plain.step(tok, pos)
    assert float((got - other).abs().max()) > 0.1 * float(other.abs().max())


def test_tree_step_follows_the_branches():
    """Every path from the root gives the logits of a chain of its tokens."""
    say("tree step branches")
    b, start = 2, 9
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 5], device=DEV)
    paths = {3: [0, 1, 3], 4: [0, 1, 4], 6: [0, 2, 5, 6]}
    tokens, prompt = _tokens((b, 7), 1), _tokens((b, start), 2)
    lengths = torch.full((b,), start, device=DEV)

    def fresh():
        run = _runner(b, 40)
        run.tree_step(prompt, torch.zeros(b, dtype=torch.int64, device=DEV))
        return run

    got = fresh().tree_step(tokens, lengths, parents)
    for leaf, path in paths.items():
        want = fresh().tree_step(tokens[:, path], lengths)
        for at, node in enumerate(path):
            _near(got[:, node], want[:, at], f"path to {leaf}, node {node}")


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rounds(temperature):
    """Rounds of drafts: the tokens, path and lengths are verification's, and the cache
    then holds what one-token steps over the accepted tokens leave."""
    say(f"rounds temperature={temperature}")
    from polarengine_vllm.kernels import tree_decode as td
    b, n = 3, 6
    run = _runner(b, 80)
    parents = torch.tensor([-1, 0, 0, 1, 2, 3], device=DEV)
    lengths = torch.tensor([0, 0, -1], device=DEV)  # the last slot is empty
    node0 = _tokens((b,), 9)
    seqs = [[int(t)] for t in node0]
    for r in range(5):
        tokens = _tokens((b, n), 20 + r)
        tokens[:, 0] = node0
        peek = run.tree_step(tokens, lengths, parents)
        best = peek.argmax(-1)
        tokens[:, 1], tokens[:, 2] = best[:, 0], (best[:, 0] + 1) % 300
        logits = run.tree_step(tokens, lengths, parents)
        tokens[2] = -1
        u = torch.rand(b, n, generator=torch.Generator().manual_seed(r)).to(DEV)
        want = td.verify_drafts(logits, tokens, u, parents, temperature=temperature)
        before = lengths.clone()
        out, path, count = run.speculative_round(tokens, lengths, u, parents, temperature=temperature)
        for x, y in zip((out, path, count), want):
            assert x.tolist() == y.tolist(), f"round {r}"
        assert lengths.tolist() == (before + count).tolist() and int(count[2]) == 0
        if temperature == 0.0:
            assert int(count[:2].min()) >= 2  # the likeliest token was drafted
        for s in range(2):
            seqs[s] += out[s, :int(count[s])].tolist()
            node0[s] = seqs[s][-1]
    for s in range(2):  # cached: all tokens but the last
        length = int(lengths[s])
        assert length == len(seqs[s]) - 1
        ref = _runner(b, 80)
        for t in range(length):
            ref.step(torch.tensor([seqs[s][t]] * b, device=DEV), torch.tensor([t], device=DEV))
        for c, w in ((run.k_cache[:, s, ..., :length], ref.k_cache[:, s, ..., :length]),
                     (run.v_cache[:, s, :, :length], ref.v_cache[:, s, :, :length])):
            _near(c.float(), w.float(), f"cache of {s}")


def test_round_replays_from_a_graph():
    say("round from a graph")
    b, n = 2, 4
    runs = [_runner(b, 64) for _ in range(2)]
    states = [{"tokens": _tokens((b, n), 5), "lengths": torch.tensor([3, 0], device=DEV),
               "u": torch.rand(b, n, generator=torch.Generator().manual_seed(1)).to(DEV)}
              for _ in runs]

    def go(run, s):
        return run.speculative_round(s["tokens"], s["lengths"], s["u"], temperature=0.8)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        go(runs[0], states[0])  # workspaces at full size
        go(runs[1], states[1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = go(runs[0], states[0])
    torch.cuda.synchronize()
    for r in range(4):
        fresh = torch.rand(b, n, generator=torch.Generator().manual_seed(r)).to(DEV)
        for s in states:
            s["u"].copy_(fresh)
            s["tokens"].copy_(_tokens((b, n), 40 + r))
        graph.replay()
        want = go(runs[1], states[1])
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), f"replay {r}"
        assert torch.equal(states[0]["lengths"], states[1]["lengths"])
        assert torch.equal(runs[0].k_cache, runs[1].k_cache)


def test_round_without_room_in_the_cache():
    say("round without room")
    b, n, max_len = 3, 4, 20
    run = _runner(b, max_len)
    run.k_cache.normal_()
    run.v_cache.normal_()
    before = run.k_cache.clone()
    lengths = torch.tensor([max_len - n, max_len - n + 1, -1], device=DEV)
    out, path, count = run.speculative_round(_tokens((b, n)), lengths, torch.rand(b, n, device=DEV))
    assert int(count[0]) >= 1 and count[1:].tolist() == [0, 0]
    assert lengths.tolist() == [max_len - n + int(count[0]), max_len - n + 1, -1]
    assert bool((out[1:] == -1).all()) and bool((path[1:] == -1).all())
    assert torch.equal(run.k_cache[:, 1:], before[:, 1:])


def test_tree_step_refusals():
    say("tree step refusals")
    run = _runner(2, 20)
    lengths = torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="tokens"):
        run.tree_step(_tokens((3, 4)), lengths)
    with pytest.raises(ValueError, match="tokens"):
        run.tree_step(_tokens((2, 4)).int(), lengths)
    with pytest.raises(ValueError, match="nodes"):
        run.tree_step(_tokens((2, 65)), lengths)
    with pytest.raises(ValueError, match="lengths"):
        run.tree_step(_tokens((2, 4)), lengths[:1])
