"""The package with a torch older than this one: without the 8-bit types, which only the
paged cache needs, and with one tensor at a time for increment_version."""

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

OLD = """
import torch, torch.autograd.graph as graph
real = graph.increment_version
def one(tensor):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("a tensor")
    real(tensor)
graph.increment_version = one
from polarengine_vllm.kernels._calls import written
x, y = torch.zeros(2), torch.zeros(2)
with torch.inference_mode():
    z = torch.zeros(2)
before = x._version, y._version
written(x, z, y)
assert (x._version, y._version) == (before[0] + 1, before[1] + 1)
"""


def test_writes_count_where_torch_takes_one_tensor_at_a_time():
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "polarengine-vllm_amd"))
    got = subprocess.run([sys.executable, "-c", OLD], env=env, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]
