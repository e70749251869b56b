"""Root-mean-square norm after the residual's addition, with the rows as they are or quantized
for the product that follows, and its gradient.

    s = x + residual                      rounded to the residual's type, as it is stored
    y = s / sqrt(mean(s^2) + eps) * weight

The residual and the weight have x's type or f32 (a residual stream kept in f32), sums are in
f32, and equal inputs give equal bits, gradients included.  Quantized rows may differ from another
f32 form's by a step of a code: a quotient of y and its block's maximum does not depend on the root,
so exact ties of 16-bit rows (one value in some thousands) fall by how each form rounded it.  ``rms_norm`` takes part in autograd
in x, weight and residual; the gradient of ``sum`` joins in the same pass.  Rows have 1 to
16384 columns at any distance.  Arguments that do not fit raise ``ValueError``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, fp4


class Normed(NamedTuple):
    """``y`` [M, H] of x's type, ``sum`` [M, H] of the residual's (None without one)."""

    y: torch.Tensor
    sum: torch.Tensor | None


class NormedQuantized(NamedTuple):
    """``rows``: ``fp4.Rows``, or E4M3 values and their scales as ``fp8.quantize`` returns them; ``sum``
    as in ``Normed``; ``y`` where it was asked for."""

    rows: fp4.Rows | tuple[torch.Tensor, torch.Tensor]
    sum: torch.Tensor | None
    y: torch.Tensor | None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6) -> Normed:
    """Rows [M, H] (bf16, f16, f32)."""
    return Normed(*_lib.ops().rms_norm(x, weight, residual, eps))


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                      format: str = "fp8", keep: bool = False) -> NormedQuantized:
    """The same with y quantized from f32, without a rounding in between: ``format`` "fp8" (E4M3, a
    scale per 128 columns), "nvfp4" or "mxfp4" (H a multiple of 32).  ``keep``: y too, of x's type (for a router).
    For serving: inputs that require a gradient are refused."""
    out = 1 if format == "fp8" else 2 + fp4._format(format) if format in fp4.FORMATS else 0
    if not out:
        raise ValueError(f"format must be one of {sorted(['fp8', *fp4.FORMATS])}, got {format!r}")
    q, scale, total, y = _lib.ops().rms_norm_quantize(x, weight, residual, eps, out, keep)
    return NormedQuantized((q, scale) if out == 1 else fp4.Rows(q, x.shape[1], format), total, y)


def rms_norm_grad(s: torch.Tensor, grad_y: torch.Tensor, weight: torch.Tensor, grad_sum: torch.Tensor | None = None,
                  eps: float = 1e-6, need_x: bool = True, need_residual: bool = True, need_weight: bool = True):
    """Gradients of ``rms_norm`` in x (``grad_y``'s type), residual (``s``'s type) and weight, None where not
    needed (one tensor for x and residual where they have one type); ``s``: the stored sum, or x where
    there was no residual."""
    return _lib.ops().rms_norm_grad(s, grad_y, grad_sum, weight, eps, need_x, need_residual, need_weight)
