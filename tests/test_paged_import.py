"""The package without the 8-bit types: they came to torch later than what the quantized
linears need, whose import must not ask for them."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import torch
del torch.float8_e8m0fnu
import polarengine_vllm.linear_method
import polarengine_vllm.decode_runner
from polarengine_vllm.kernels import polar_gemm, tree_attention, token_logprobs, new_cache
try:
    new_cache(4, 2, 16, 64, "cpu")
except RuntimeError as e:
    assert "float8_e8m0fnu" in str(e), e
else:
    raise SystemExit("a cache without its type")
"""


def test_import_without_the_scales_type():
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "polarengine-vllm_amd"))
    got = subprocess.run([sys.executable, "-c", CODE], env=env, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]
