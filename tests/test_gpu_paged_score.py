"""GPU tests of DecodeRunner.score with the tokens that follow a step's rows: a prompt that
is scored chunk by chunk has a log probability for every token."""

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_paged_cache import _i64
from test_gpu_tree_runner import _runner, _tokens

pytestmark = pytest.mark.gpu


def test_a_chunks_last_row_scores_the_token_behind_it():
    say("paged runner scores, chunk by chunk")
    from polarengine_vllm.kernels.logprobs import token_logprobs
    run, same = _runner(1, 128), _runner(1, 128)
    pools = [r.paged_pool(blocks=30, batch=4, block_size=16) for r in (run, same)]
    for p in pools:
        p.keep(_i64([0, 0, -1, 0]).to(DEV))
    for step, (counts, follow) in enumerate([([20, 0, 9, 17], [7, 8, 9, 1 << 40]), ([1, 30, 0, 1], [3, -1, 5, 6]),
                                             ([0, 0, 0, 45], [1, 2, 3, 4])]):
        tokens, c, f = _tokens((45,), step), _i64(counts).to(DEV), _i64(follow).to(DEV)
        out = run.score(tokens, c, pools[0], top=3, follow=f)
        _, attend = same._paged(tokens, c, pools[1], None, 0)
        logits = same._layers(tokens, attend)
        want, row = [-1] * 45, 0
        for b, n in enumerate(counts):
            n = 0 if b == 2 else n  # an empty slot
            want[row:row + n] = tokens.tolist()[row + 1:row + n] + [follow[b]] if n else []
            row += n
        for name, got, w in zip(out._fields, out, token_logprobs(logits, _i64(want).to(DEV), 3)):
            assert torch.equal(got, w), name
    lengths = pools[0].lengths.tolist()
    with pytest.raises((TypeError, ValueError)):
        run.score(tokens, c, pools[0], follow=f[:3])
    with pytest.raises((TypeError, ValueError)):
        run.score(tokens, c, pools[0], follow=f.int())
    assert pools[0].lengths.tolist() == lengths


def test_captured_score():
    run, same = _runner(1, 128), _runner(1, 128)
    pools = [r.paged_pool(blocks=30, batch=2, block_size=16) for r in (run, same)]
    scratch = run.paged_pool(blocks=30, batch=2, block_size=16)
    for p in pools:
        p.keep(_i64([0, 0]).to(DEV))
    tokens, counts, follow = _tokens((12,), 1), _i64([5, 7]).to(DEV), _i64([3, 4]).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run.score(tokens, counts, scratch, 2, follow=follow)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run.score(tokens, counts, pools[0], 2, follow=follow)
    torch.cuda.synchronize()
    for i in range(5):
        say(f"score replay {i}")
        tokens.copy_(_tokens((12,), 10 + i)), counts.copy_(_i64([[5, 7], [0, 3], [12, 0], [1, 1], [6, 6]][i]))
        follow.add_(1)
        graph.replay()
        want = same.score(tokens, counts, pools[1], 2, follow=follow)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
