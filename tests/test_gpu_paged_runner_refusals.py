"""GPU tests of DecodeRunner over a paged cache: a call that is refused has changed nothing,
neither the pool's lengths, tables and stack nor its caches."""

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_paged_cache import _i64
from test_gpu_tree_runner import _runner, _tokens

pytestmark = pytest.mark.gpu


def _state(pool):
    parts = [pool.lengths, pool.tables, pool.free, pool.free_count]
    for cache in pool.caches:
        parts += [x.view(torch.uint8) for x in cache]
    return [x.clone() for x in parts]


def test_a_refused_step_leaves_the_pool():
    from polarengine_vllm.kernels.paged_cache import PagedPool
    run = _runner(1, 64)
    c = run.cfg
    pool = run.paged_pool(blocks=8, batch=2, block_size=16)
    pool.keep(_i64([0, 0]).to(DEV))
    tokens, counts = _tokens((9,), 1), _i64([4, 5]).to(DEV)
    run.paged_step(tokens, counts, pool)
    heads, dims = [PagedPool(c.layers, 8, h, d, 2, 64, DEV, 16) for h, d in ((c.kv_heads + 1, c.head_dim),
                                                                            (c.kv_heads, 256))]
    assert c.head_dim != 256
    for p in (heads, dims):
        p.keep(_i64([0, 0]).to(DEV))
    calls = {
        "window": lambda: run.paged_step(tokens, counts, pool, window=0),
        "sinks": lambda: run.paged_step(tokens, counts, pool, window=3, sinks=-1),
        "score's window": lambda: run.score(tokens, counts, pool, window=-2),
        "top": lambda: run.score(tokens, counts, pool, top=65),
        "top below 0": lambda: run.score(tokens, counts, pool, top=-1),
        "tokens of another device": lambda: run.paged_step(tokens.cpu(), counts, pool),
        "counts of another device": lambda: run.paged_step(tokens, counts.cpu(), pool),
        "counts of another type": lambda: run.paged_step(tokens, counts.int(), pool),
        "heads": lambda: run.paged_step(tokens, counts, heads),
        "head_dim": lambda: run.paged_step(tokens, counts, dims),
    }
    before = [_state(p) for p in (pool, heads, dims)]
    for name, call in calls.items():
        say(f"refused: {name}")
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
        torch.cuda.synchronize()
        for p, was in zip((pool, heads, dims), before):
            for a, b in zip(_state(p), was):
                assert torch.equal(a, b), name
    run.paged_step(tokens, counts, pool)  # and the pool goes on
    assert pool.lengths.tolist() == [8, 10]


def test_numbers_that_are_not_whole_leave_the_pool():
    run = _runner(1, 64)
    pool = run.paged_pool(blocks=8, batch=2, block_size=16)
    pool.keep(_i64([0, 0]).to(DEV))
    tokens, counts = _tokens((9,), 1), _i64([4, 5]).to(DEV)
    run.paged_step(tokens, counts, pool)
    before = _state(pool)
    for name, call in {"window": lambda: run.paged_step(tokens, counts, pool, window=8.0),
                       "sinks": lambda: run.paged_step(tokens, counts, pool, window=8, sinks=1.0),
                       "top": lambda: run.score(tokens, counts, pool, top=3.0)}.items():
        say(f"refused: {name} as a float")
        with pytest.raises(TypeError):
            call()
        torch.cuda.synchronize()
        for a, b in zip(_state(pool), before):
            assert torch.equal(a, b), name
