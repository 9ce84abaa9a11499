"""GPU tests of the norm + rotary kernel's one rounding: every value is the 64-bit
formula's rounded once to 16 bits, unless that lies within 2^-40 of its size of the
middle between two (the 64-bit arithmetic itself is good to 2^-45)."""

import numpy as np
import pytest
import torch

import test_gpu_tree_decode as base
from gpu_helpers import DEV, say

pytestmark = pytest.mark.gpu


def _round_once(y, dtype):
    """float64 y rounded once to the type (normal range), and whether it is clear of the
    middles: significands of p bits, to nearest, ties to even."""
    p = 11 if dtype is torch.float16 else 8
    m, e = np.frexp(y)
    m = m * 2.0 ** p
    r = np.rint(m)
    clear = np.abs(np.abs(m - np.floor(m)) - 0.5) > 2.0 ** (p - 40)
    return np.ldexp(r, e - p), clear & (np.abs(y) >= torch.finfo(dtype).smallest_normal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("heads,kv,dim,rot", [(14, 2, 128, 128), (6, 1, 64, 64), (3, 2, 256, 96)])
def test_values_are_rounded_once(dtype, norm, heads, kv, dim, rot):
    say(f"norm_rope rounding {dtype} norm={norm} heads={heads}/{kv} dim={dim} rot={rot}")
    rows, g = 600, torch.Generator().manual_seed(dim + rot)
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).to(dtype)
    ang = torch.rand(rows, rot // 2, generator=g, dtype=torch.float64) * 6.28
    table = torch.cat([ang.cos(), ang.sin()], 1).float()
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype) if norm else None
    pos = torch.randperm(rows, generator=g)
    wd = None if w is None else w.to(DEV)
    got = base._td().qk_norm_rope(qkv.to(DEV), heads, kv, table.to(DEV), pos.to(DEV), wd, wd, base.EPS)
    eps, base_eps = float(np.float32(base.EPS)), base.EPS  # eps passes through fp32
    try:
        base.EPS = eps
        ref = base._rope_ref(qkv, heads, kv, table, pos, w, w)
    finally:
        base.EPS = base_eps
    for x, (want, _), what in zip(got, ref, "qk"):
        once, clear = _round_once(want.numpy(), dtype)
        have = x.double().cpu().numpy()
        bad = (have != once) & clear
        assert clear.mean() > 0.99 and not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}"
