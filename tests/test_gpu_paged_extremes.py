"""GPU tests of paged attention over values at the ends of their 16-bit types: a mean of
finite values is finite. Tolerances and reference are those of test_gpu_paged_scales."""

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_paged_scales import _case, _compare, _i64, _pc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,group,d,lengths", [(1, 4, 128, [300]), (1, 4, 64, [9000, 40]), (2, 4, 256, [5000]),
                                                 (40, 8, 128, [500]), (64, 4, 64, [3000]), (40, 4, 256, [900, 70])])
def test_largest_values(new, group, d, lengths, dtype):
    """Values as the write puts them into the cache, up to 0.99 of the largest number."""
    pc = _pc()
    say(f"largest values {new} x {group} x {d} {lengths} {dtype}")
    t = 32
    q, cache, tables, starts, lengths = _case(d, len(lengths), 2, group, d, t, dtype, [new] * len(lengths), lengths)
    g = torch.Generator().manual_seed(3)
    dev = pc.PagedCache(*(x.to(DEV) for x in cache))
    for b, n in enumerate(lengths):
        k = torch.randn(n, 2, d, generator=g).to(dtype)
        u = torch.rand(n, 2, d, generator=g) * 2 - 1
        v = (u.sign() * u.abs().clamp(min=0.5) * 0.99 * torch.finfo(dtype).max).to(dtype)
        if b == 0:
            v = v.abs()  # no cancelling: the mean is as large
        slots = [tables[b][j // t] * t + j % t for j in range(n)]
        pc.write_blocks(k.to(DEV), v.to(DEV), dev, _i64(slots).to(DEV))
    host = pc.PagedCache(*(x.cpu() for x in dev))
    got = _compare((q, host, tables, starts, lengths))
    assert float(got.abs().max()) > 0.5 * torch.finfo(dtype).max
