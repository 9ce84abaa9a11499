"""CPU tests of PagedPool's book-keeping of lengths: the library's calls are left out."""

import torch


def test_keep_begins_a_sequence_with_0_alone(monkeypatch):
    """An empty slot stays empty where positions are to stay that it does not have."""
    from polarengine_vllm.kernels import paged_cache as pc
    kept = []
    monkeypatch.setattr(pc, "release_blocks", lambda tables, keep, *rest: kept.append(keep.tolist()))
    pool = pc.PagedPool(1, 8, 2, 64, 6, 64, "cpu", block_size=16)
    pool.lengths.copy_(torch.tensor([-1, -1, -1, 20, 20, 20]))
    pool.keep(torch.tensor([1 << 40, 1, 0, 1 << 40, 0, -1]))
    assert pool.lengths.tolist() == [-1, -1, 0, 20, 0, -1]
    pool.keep(pool.lengths)  # everything as it is
    assert pool.lengths.tolist() == [-1, -1, 0, 20, 0, -1]
    assert kept == [[1 << 40, 1, 0, 1 << 40, 0, 0], [0, 0, 0, 20, 0, 0]]
