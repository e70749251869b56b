"""What the stateless operators (``permute``, ``fp8``) share: argument checks, the
current stream, and the device's operator error word."""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib

DTYPE_CODE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.FP32}
_HERE = contextlib.nullcontext()


def stream(device: torch.device) -> int:
    """Handle of torch's current stream on ``device``."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def on(device: torch.device):
    """Makes ``device`` current for a launch (free where it is already)."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def empty(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A contiguous matrix (the strided call parses its arguments in two thirds of ``torch.empty``'s time)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def want(name: str, t: torch.Tensor, dtypes, dim: int, device: torch.device | None = None, rows: bool = False) -> None:
    """``t`` is a CUDA tensor of one of ``dtypes`` with ``dim`` axes, contiguous or
    (``rows``) with any distance between rows, on ``device`` when given."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor, got {getattr(t, 'device', type(t))}")
    if t.dtype not in dtypes or t.dim() != dim:
        raise ValueError(f"{name} must be {'/'.join(str(d) for d in dtypes)} with {dim} axes, got {t.dtype} "
                         f"{tuple(t.shape)}")
    if not t.is_contiguous() and not (rows and t.stride(-1) == 1 and t.stride(0) >= t.shape[1]):
        raise ValueError(f"{name} must {'have contiguous rows' if rows else 'be contiguous'}, got strides {t.stride()}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other arguments on {device}")


def want_shape(name: str, t: torch.Tensor, shape) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def check_errors(device: torch.device | int | None = None) -> None:
    """Wait for ``device``'s current stream and raise if an operator found a row or
    offset out of range (or a wait ran out) since the last check."""
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else
                       (device if isinstance(device, int) else torch.device(device).index))
    bits = ctypes.c_uint32(0)
    with on(dev):
        _lib.check("operators", _lib.lib().b200moe_op_errors(stream(dev), ctypes.byref(bits)))
