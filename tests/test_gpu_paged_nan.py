"""GPU tests of paged attention with NaN codes at a few places: the rows that see one, and
no others, are NaN (of a value, in its dimension). Reference and tolerances are those of
test_gpu_paged_cache."""

import random

import pytest
import torch

from gpu_helpers import DEV, say
from test_gpu_paged_cache import _attend_compare
from test_gpu_paged_scales import FORMS, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,group,d", FORMS)
@pytest.mark.parametrize("t", [16, 64])
def test_few_nan(new, group, d, t):
    rng = random.Random(new * d + t)
    dtype = rng.choice([torch.bfloat16, torch.float16])
    lengths = [new + 60, 250, 390]
    for trial in range(3):
        say(f"few NaN {new} x {group} x {d} blocks of {t} {dtype} trial {trial}")
        case = _case(d + trial, 3, 2, group, d, t, dtype, [new] * 3, lengths)
        q, cache, tables, starts, _ = case
        k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
        for b, n in enumerate(lengths):
            if n % t:  # memory that nothing has written
                k[tables[b][n // t], :, n % t:], v[tables[b][n // t], :, :, n % t:] = 0xFF, 0x7F
            places = [n - 1 - rng.randrange(new) for _ in range(2)] + [rng.randrange(n) for _ in range(3)]
            for j in places:  # one dimension, or all of some, of one head's values
                dims = rng.choice([[rng.randrange(d)], range(d // 2), range(d // 2, d), range(d)])
                v[tables[b][j // t], rng.randrange(2), list(dims), j % t] = rng.choice([0x7F, 0xFF])
            if trial == 2:
                j = rng.choice(places)
                k[tables[b][j // t], rng.randrange(2), j % t, rng.randrange(d)] = 0x7F
        _attend_compare(case)
        _attend_compare(case, rng.choice([20, 64, 130]), rng.choice([0, 3, 17]))
