"""What :mod:`shipinfer_b200.logprobs` and :mod:`shipinfer_b200.routing` share: the checks of
their tensors, and the device and stream that a call runs on."""

from __future__ import annotations

from contextlib import nullcontext
from typing import Any

from shipinfer_b200 import _native
from shipinfer_b200.errors import ConfigurationError, ValidationError


def _torch():
    import torch

    return torch


def element_code(t: Any, name: str) -> int:
    """The C ABI's code of a score or result tensor's type."""
    torch = _torch()
    code = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16,
            torch.bfloat16: _native.DTYPE_BF16}.get(t.dtype)
    if code is None:
        raise ValidationError(f"{name} must be float32, float16 or bfloat16; got {t.dtype}")
    return code


def small(value: Any, name: str) -> int:
    """An integer that the C ABI takes as 32 bits: one that does not fit would arrive as another."""
    value = int(value)
    if not -(1 << 31) <= value < 1 << 31:
        raise ConfigurationError(f"{name} {value} does not fit in 32 bits")
    return value


def check_matrix(t: Any, name: str) -> tuple[int, int]:
    """A score or result matrix: its rows may lie apart, the values within one may not."""
    if t.dim() != 2:
        raise ValidationError(f"{name} must have two dimensions; got {tuple(t.shape)}")
    rows, cols = small(t.shape[0], f"{name} rows"), small(t.shape[1], f"{name} columns")
    if cols > 1 and rows > 0 and int(t.stride(1)) != 1:
        raise ValidationError(f"{name}: the values of a row must be adjacent; strides {tuple(t.stride())}")
    if t.requires_grad and _torch().is_grad_enabled():
        raise ValidationError(f"{name} asks for a gradient; this call computes none (use no_grad or detach)")
    return rows, cols


def check_dense(t: Any, name: str, dtype: Any, shape: tuple[int, ...]) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValidationError(
            f"{name} must be a contiguous {str(dtype).removeprefix('torch.')} {list(shape)} CUDA tensor; "
            f"got {t.dtype} {list(t.shape)}"
        )


def check_device(like: Any, **others: Any) -> Any:
    """The CUDA device that every tensor of the call is on."""
    for name, t in others.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValidationError(f"{name} must be a CUDA tensor; it is on {t.device}")
        if t.device != like.device:
            raise ValidationError(f"{name} is on {t.device}, another tensor of the call on {like.device}")
    return like.device


def guard(device: Any) -> Any:
    torch = _torch()
    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def handle_of(device: Any, stream: int | None) -> int:
    """The launch's stream: the one given, else torch's current stream on the device."""
    return int(_torch().cuda.current_stream(device).cuda_stream) if stream is None else int(stream)


def empty(shape: tuple[int, ...], dtype: Any, device: Any, stream: int | None) -> Any:
    """A result of the call, allocated on the stream that writes it."""
    torch = _torch()
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    on = torch.cuda.ExternalStream(int(stream), device=device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(on):
        return torch.empty(shape, dtype=dtype, device=device)


def ptr(t: Any) -> int | None:
    return t.data_ptr() if t is not None and t.numel() else None
