"""What :mod:`shipinfer_b200.logprobs` and :mod:`shipinfer_b200.routing` share: the checks of
their tensors, and the device and stream that a call runs on."""

from __future__ import annotations

from contextlib import nullcontext
from typing import Any

import torch
from torch.autograd import forward_ad

from shipinfer_b200 import _native
from shipinfer_b200.errors import ConfigurationError, ValidationError

_CODES = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}
_SAME_DEVICE = nullcontext()
#: torch's current stream on a device as a handle, without the stream object that
#: torch.cuda.current_stream() builds around it (2 us of a call whose kernel takes 3)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def element_code(t: Any, name: str) -> int:
    """The C ABI's code of a score or result tensor's type."""
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValidationError(f"{name} must be float32, float16 or bfloat16; got {t.dtype}")
    return code


def small(value: Any, name: str) -> int:
    """A whole number that the C ABI takes as 32 bits: one that does not fit would arrive as another."""
    given = value
    try:
        value = int(given)
    except (TypeError, ValueError, OverflowError):
        value = None
    if value is None or value != given:
        raise ValidationError(f"{name} must be a whole number; got {given!r}")
    if not -(1 << 31) <= value < 1 << 31:
        raise ConfigurationError(f"{name} {value} does not fit in 32 bits")
    return value


def refuse_gradient(t: Any, name: str) -> None:
    """A result without its gradient or tangent would pass for one that does not depend on `t`."""
    # outside every dual level (-1), where no tensor has a tangent, unpack_dual's 0.5 us are spared
    if (t.requires_grad and torch.is_grad_enabled()) or (
        getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None
    ):
        raise ValidationError(f"{name} asks for a gradient; this call computes none (use no_grad, detach or the primal)")


def check_matrix(t: Any, name: str) -> tuple[int, int]:
    """A score or result matrix: its rows may lie apart, the values within one may not."""
    if t.dim() != 2:
        raise ValidationError(f"{name} must have two dimensions; got {tuple(t.shape)}")
    rows, cols = t.shape
    if rows >= 1 << 31 or cols >= 1 << 31:
        raise ConfigurationError(f"{name}: {rows} rows of {cols} do not fit in 32 bits")
    if cols > 1 and rows > 0 and t.stride(1) != 1:
        raise ValidationError(f"{name}: the values of a row must be adjacent; strides {tuple(t.stride())}")
    refuse_gradient(t, name)
    return rows, cols


def check_dense(t: Any, name: str, dtype: Any, shape: tuple[int, ...]) -> None:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValidationError(
            f"{name} must be a contiguous {str(dtype).removeprefix('torch.')} {list(shape)} CUDA tensor; "
            f"got {t.dtype} {list(t.shape)}"
        )
    refuse_gradient(t, name)


def check_device(*tensors: Any) -> int:
    """The CUDA device that every tensor of the call is on (``None``: not given)."""
    index = tensors[0].get_device()
    if index < 0:
        raise ValidationError(f"the tensors of the call must be CUDA tensors; one is on {tensors[0].device}")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValidationError(f"a tensor of the call is on {t.device}, another on cuda:{index}")
    return index


def guard(index: int) -> Any:
    return _SAME_DEVICE if _get_device() == index else torch.cuda.device(index)


def handle_of(index: int, stream: int | None) -> int:
    """The launch's stream: the one given, else torch's current stream on the device."""
    if stream is not None:
        return int(stream)
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def empty(shape: tuple[int, ...], dtype: Any, index: int, stream: int | None) -> Any:
    """A result of the call, allocated on the stream that writes it."""
    device = torch.device("cuda", index)
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    on = torch.cuda.ExternalStream(int(stream), device=device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(on):
        return torch.empty(shape, dtype=dtype, device=device)


def ptr(t: Any) -> int | None:
    return None if t is None else t.data_ptr()  # 0, a null pointer, for an empty tensor
