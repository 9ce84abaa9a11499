"""What the operators around the quantized linears share: calls into the library and
the checks of what they are given."""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.graph import increment_version

from polarengine_vllm import _lib

try:
    increment_version(())  # several at once, 0.9 against 2.2 us for four
    _count = increment_version
except TypeError:  # an older torch takes one tensor

    def _count(tensors) -> None:
        for t in tensors:
            increment_version(t)


def call(name: str, dev: torch.device, *args) -> None:
    """One call into the library on the device's current stream, the device made the
    current one around it where it is another."""
    lib = _lib.lib()
    here, index = torch._C._cuda_getDevice(), dev.index
    if here == index:
        rc = getattr(lib, name)(*args, _lib.stream_ptr(dev))
    else:
        torch._C._cuda_setDevice(index)
        try:
            rc = getattr(lib, name)(*args, _lib.stream_ptr(dev))
        finally:
            torch._C._cuda_setDevice(here)
    if rc:
        _lib.check(rc, name)


def inputs(*tensors: Optional[torch.Tensor]) -> torch.device:
    """The one GPU of the tensors; refuses others, and inputs that autograd follows
    (reverse mode, or forward mode, which no_grad does not turn off)."""
    grad = torch.is_grad_enabled()
    dual = fwAD._current_level >= 0  # outside a dual level no tensor has a tangent
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None:
            if t.get_device() != index or index < 0:
                _lib.require_device(*tensors)
            if (grad and t.requires_grad) or (
                    dual and not t.is_inference() and fwAD.unpack_dual(t).tangent is not None):
                raise RuntimeError("the kernels of drafted tokens, the paged cache and log "
                                   "probabilities have no backward pass: call them under "
                                   "torch.no_grad(), without forward-mode tangents, or detach "
                                   "their inputs")
    return tensors[0].device


def int64(t: torch.Tensor, shape: Tuple[int, ...], name: str) -> torch.Tensor:
    if t.dtype is not torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t.contiguous()


def written(*tensors: torch.Tensor) -> None:
    """Counts writes through raw pointers (inference tensors keep no count)."""
    if any(t.is_inference() for t in tensors):
        tensors = tuple(t for t in tensors if not t.is_inference())
    _count(tensors)
