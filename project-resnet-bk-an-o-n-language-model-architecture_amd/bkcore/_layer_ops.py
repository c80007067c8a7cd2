"""Argument handling shared by the mixing layer's operators (norm, convolution, selective scan, attention)."""
from __future__ import annotations

import torch

from . import _lib
from .bk_core import _on_device as on_device

DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def need_device(first: torch.Tensor, *others) -> None:
    """All given tensors (None is skipped) on the ROCm device of the first one."""
    for t in (first, *others):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("bkcore: tensors must be on a ROCm device (no CPU path)")
        if t.device != first.device:
            raise RuntimeError(f"bkcore: tensors on different devices ({first.device} and {t.device})")


def need_dtype(what: str, first: torch.Tensor, *others) -> int:
    """The library's code of the common element type."""
    if first.dtype not in DTYPES:
        raise TypeError(f"bkcore: {what} takes float32, bfloat16 or float16 tensors, not {first.dtype}")
    for t in others:
        if t is not None and t.dtype != first.dtype:
            raise TypeError(f"bkcore: {what} takes operands of one type, got {first.dtype} and {t.dtype}")
    return DTYPES[first.dtype]


def need_param(what: str, p: torch.Tensor | None, x: torch.Tensor) -> None:
    if p is not None and p.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"bkcore: {what}: parameters are float32 or of the input's type {x.dtype}, not {p.dtype}")


def need_shape(what: str, name: str, t: torch.Tensor | None, shape: tuple) -> None:
    if t is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"bkcore: {what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def need_state(what: str, name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    """A buffer that the call updates in place."""
    need_shape(what, name, t, shape)
    if t.dtype != dtype:
        raise TypeError(f"bkcore: {what}: {name} is {t.dtype}, expected {dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"bkcore: {what} updates {name} in place and keeps no gradient; detach it or use torch.no_grad()")


def no_grad_through(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"bkcore: {what} serves single tokens and has no gradient; call it under torch.no_grad()")


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def lengths_arg(what: str, lengths: torch.Tensor | None, x: torch.Tensor, batch: int, longest: int):
    """(B,) lengths as int32 on x's device."""
    if lengths is None:
        return None
    need_shape(what, "lengths", lengths, (batch,))
    need_device(x, lengths)
    if lengths.dtype == torch.int32:
        return lengths.contiguous()
    if lengths.dtype != torch.int64:
        raise TypeError(f"bkcore: {what}: lengths are int32 or int64, not {lengths.dtype}")
    return lengths.clamp(0, longest).to(torch.int32)


def stream(index: int) -> int:
    """The current stream's handle on a device, without a Stream object around it."""
    return torch._C._cuda_getCurrentRawStream(index)
