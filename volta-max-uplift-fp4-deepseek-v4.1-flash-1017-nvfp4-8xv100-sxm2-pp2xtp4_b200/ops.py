"""What the stateless operators (``permute``, ``fp8``, ``fp4``, ``norm``) share: their binding and the
device's operator error word.

Gradients are of first order and reverse mode: a second differentiation and a tensor
with a forward-mode tangent (``torch.autograd.forward_ad``) raise ``NotImplementedError``."""

from __future__ import annotations

import ctypes

import torch

from . import _lib


def check_errors(device: torch.device | int | None = None) -> None:
    """Wait for ``device``'s current stream and raise if an operator found a row or
    offset out of range (or a wait ran out) since the last check."""
    index = device if isinstance(device, int) else None if device is None else torch.device(device).index
    with torch.cuda.device(torch.cuda.current_device() if index is None else index):
        bits = ctypes.c_uint32(0)
        _lib.check("operators", _lib.lib().b200moe_op_errors(torch.cuda.current_stream().cuda_stream,
                                                             ctypes.byref(bits)))
