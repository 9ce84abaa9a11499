"""gfx950 kernels behind the reference's kernel-module names."""

from polarengine_vllm.kernels.fwht import FWHTCache, build_hadamard, fwht_matmul, fwht_pairs
from polarengine_vllm.kernels.polar_gemm import polar_gemm, polar_gemm_packed, polar_matmul
from polarengine_vllm.kernels.polar_gemv import pack_codes_int4, polar_gemv, polar_gemv_packed
from polarengine_vllm.kernels.polar_gemv_splitk import polar_gemv_packed_splitk, polar_gemv_splitk
from polarengine_vllm.kernels.tree_decode import (
    TreePlan, keep_accepted, qk_norm_rope, qk_norm_rope_write, tree_attention, tree_plan,
    verify_drafts)

__all__ = [
    "FWHTCache", "build_hadamard", "fwht_matmul", "fwht_pairs",
    "polar_gemm", "polar_gemm_packed", "polar_matmul",
    "pack_codes_int4", "polar_gemv", "polar_gemv_packed",
    "polar_gemv_packed_splitk", "polar_gemv_splitk",
    "TreePlan", "keep_accepted", "qk_norm_rope", "qk_norm_rope_write", "tree_attention",
    "tree_plan", "verify_drafts",
]
