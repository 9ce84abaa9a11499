"""Log probabilities of given tokens (no reference file: vLLM's sampler plays this
part there): what a server answers beside its tokens, and how a prompt is scored.

There is no backward pass: inputs that autograd follows are refused.
"""

from __future__ import annotations

from operator import index
from typing import NamedTuple

import torch

from polarengine_vllm import _lib
from polarengine_vllm.kernels._calls import call, inputs, int64

MAX_TOP = 64
_DTYPES = {torch.float16: _lib.PE_DTYPE_F16, torch.bfloat16: _lib.PE_DTYPE_BF16,
           torch.float32: _lib.PE_DTYPE_F32}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # float32 [rows]: log softmax(logits) at the row's token
    rank: torch.Tensor          # int64 [rows]: tokens before it, 0 for the likeliest
    entropy: torch.Tensor       # float32 [rows]: of softmax(logits)
    top_logprobs: torch.Tensor  # float32 [rows, top]: of the likeliest tokens, in order
    top_tokens: torch.Tensor    # int64 [rows, top]


def check_top(top: int, vocab: int) -> None:
    """Refuses a number of alternatives that ``token_logprobs`` has none for."""
    if not 0 <= index(top) <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, vocab)}, got {top}")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Of logits [rows, vocab] (fp32, fp16 or bf16; -inf where a token is ruled out) and
    tokens int64 [rows] (outside the vocabulary: none, with logprob 0 and rank -1).
    Equal logits rank by number. ``top``: 0 to 64, at most the vocabulary. A NaN counts as
    -inf; ruled-out tokens have logprob -inf and follow the others by number. A row with
    +inf, or without a finite logit, has no distribution: its numbers say nothing."""
    dev = inputs(logits, tokens)
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if logits.dim() != 2 or not logits.shape[1]:
        raise ValueError(f"logits must be [rows, vocab], got {list(logits.shape)}")
    rows, vocab = logits.shape
    check_top(top, vocab)
    tokens = int64(tokens, (rows,), "tokens")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    f32, i64 = torch.float32, torch.int64
    out = TokenLogprobs(torch.empty(rows, dtype=f32, device=dev), torch.empty(rows, dtype=i64, device=dev),
                        torch.empty(rows, dtype=f32, device=dev),
                        torch.empty(rows, top, dtype=f32, device=dev),
                        torch.empty(rows, top, dtype=i64, device=dev))
    if not rows:
        return out
    size = _lib.workspace_size("pe_token_logprobs_workspace_size", rows, vocab, top)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    call("pe_token_logprobs", dev, logits.data_ptr(), code, rows,
         logits.stride(0) if rows > 1 else vocab, vocab, tokens.data_ptr(), top,
         out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), out[4].data_ptr(),
         _lib.ptr(ws), size)
    return out
