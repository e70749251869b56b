"""8-bit floating point (E4M3) products with a scale for each block of 128.

Activations carry a scale per row and 128 columns, weights one per 128 x 128 block:

    amax = max(max |x|, 1e-30)    scale = amax / 448    q = e4m3(x * (448 / amax))

A NaN or an infinity in a block makes the whole block, and so its product's row,
NaN.  Products sum in f32.  Weights are frozen: ``linear`` has a gradient in its rows (a
second product, of the quantized gradient with the transposed weights), never in
the packed weights.  The quantizers, ``matmul`` and ``grouped_matmul`` return values
without a graph; ``experts.Fp8Experts`` puts the gradients of the whole path together.
Arguments that do not fit raise ``ValueError`` (an address off
16 bytes ``B200MoeError``); offsets out of range are cut and reported by
``check_errors``.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import check_errors  # noqa: F401

BLOCK = 128


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (bf16, f16, f32) -> (E4M3 [M, K], scale f32 [M, ceil(K / 128)])."""
    return _lib.ops().quantize(x)


def swiglu_quantize(h: torch.Tensor, limit: float | None = 10.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Limited SwiGLU of rows [M, 2 I] (gate columns, then up), quantized:
    ``g / (1 + exp(-g)) * u`` with ``g = min(gate, limit)``, ``u = clamp(up, -limit, limit)``,
    each step one f32 operation (a gate of -inf or a type's lowest value gives 0)."""
    return _lib.ops().swiglu_quantize(h, limit)


def swiglu_grad(h: torch.Tensor, grad: torch.Tensor, limit: float | None = 10.0) -> torch.Tensor:
    """Gradient of the SwiGLU in ``h`` [M, 2 I] for ``grad`` [M, I] of its output (the
    quantizer passes it on unchanged); zero where a bound cut the value."""
    return _lib.ops().swiglu_grad(h, grad, limit)


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights [N, K] or [E, N, K] (bf16, f16, f32) -> (E4M3 of the same shape, scale f32
    [(E,) ceil(N / 128), ceil(K / 128)])."""
    return _lib.ops().quantize_weight(w)


def transpose_weight(w: torch.Tensor, w_scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Packed weights [(E,) N, K] -> [(E,) K, N] with their blocks' scales: the weights
    of the product that gives the activations' gradient."""
    return _lib.ops().transpose_weight(w, w_scale)


def matmul(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[M, N] = quantized rows [M, K] times packed weights [N, K] transposed (K a multiple of 16)."""
    return _lib.ops().matmul(q, scale, w, w_scale, out_dtype)


def grouped_matmul(q: torch.Tensor, scale: torch.Tensor, offsets: torch.Tensor, w: torch.Tensor,
                   w_scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Rows sorted by expert (``permute``) times each expert's weights [E, N, K]: rows
    ``offsets[e] : offsets[e + 1]`` use ``w[e]``; rows before ``offsets[0]`` and from ``offsets[E]``
    on become zeros.  Offsets that fall or pass the rows are reported; those experts have no result, nor
    have later ones that go back over an earlier one's rows."""
    return _lib.ops().grouped_matmul(q, scale, offsets, w, w_scale, out_dtype)


def linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, wt: torch.Tensor | None = None,
           wt_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x`` [M, K] (bf16, f16, f32) quantized and multiplied with packed weights [N, K]
    transposed; ``out_dtype`` defaults to x's.  Where x needs a gradient (N a multiple of
    16 then), pass ``transpose_weight``'s result as ``wt`` / ``wt_scale`` to save its
    making in each backward pass."""
    return _lib.ops().linear(x, w, w_scale, wt, wt_scale, out_dtype)
