"""4-bit floating point (E2M1) rows and weights with a scale per block, and their products.

    NVFP4: 16 columns share an E4M3 scale, a row (of activations) or a matrix (of weights)
           an f32 factor, the smallest 2^e with 2688 * 2^e >= max |x| (at least 2^-100):
           scale = e4m3(max |x| / (6 factor)),  q = e2m1(x / (scale * factor))
    MXFP4: 32 columns share a scale 2^e, the smallest with 6 * 2^e >= max |x|: q = e2m1(x / 2^e)

Roundings go to nearest, ties to even, and end at 6.  A NaN or an infinity makes a row's
factor (NVFP4) or a block's scale (MXFP4) a NaN, and so its product's row.  Products take
both operands in the same format, sum in f32 and round once.  Weights are ``quantize_weight``'s or a
pack's: ``Weights(*packing.quantize_nvfp4(w))``, ``Weights(*packing.quantize_mxfp4(w))``.

For serving: rows that require a gradient are refused (``quantize``, ``swiglu_quantize``, ``linear``) but
under ``torch.no_grad``, and values come back without a graph.  Columns come in multiples of 32.  Arguments that do not fit raise ``ValueError`` (a
packed operand's address off 16 bytes ``B200MoeError``); offsets out of range are cut and reported by
``check_errors``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ops import check_errors  # noqa: F401
from .permute import permute as _permute

FORMATS = {"nvfp4": _lib.NVFP4, "mxfp4": _lib.MXFP4}


def _format(name: str) -> int:
    if name not in FORMATS:
        raise ValueError(f"format must be one of {sorted(FORMATS)}, got {name!r}")
    return FORMATS[name]


class Rows(NamedTuple):
    """Quantized rows.  ``record`` uint8 [M, R] holds a row's codes (``columns`` / 2 bytes, the
    even column in the low bits), its scales, for NVFP4 on the next multiple of four its
    factor, and zeros up to a multiple of 16 bytes."""

    record: torch.Tensor
    columns: int
    format: str

    @property
    def codes(self) -> torch.Tensor:
        return self.record[:, : self.columns // 2]

    @property
    def scale(self) -> torch.Tensor:
        """E4M3 (NVFP4) or E8M0 (MXFP4) bytes [M, columns / 16 or / 32]."""
        n = self.columns // (16 if self.format == "nvfp4" else 32)
        return self.record[:, self.columns // 2: self.columns // 2 + n]

    @property
    def factor(self) -> torch.Tensor | None:
        """f32 [M] (NVFP4)."""
        if self.format != "nvfp4":
            return None
        at = self.columns // 2 + -(-self.columns // 64) * 4
        return self.record[:, at: at + 4].view(torch.float32)[:, 0]


class Weights(NamedTuple):
    """``codes`` uint8 [(E,) N, K / 2]; ``scale`` uint8 [(E,) N, K / 16] (E4M3) and ``factor`` f32 [E]
    ([1] for one matrix) for NVFP4, ``scale`` [(E,) N, K / 32] (E8M0) and no factor for MXFP4.  Scales have
    no sign: the products take a set sign bit of E4M3 as they like."""

    codes: torch.Tensor
    scale: torch.Tensor
    factor: torch.Tensor | None = None

    @property
    def format(self) -> str:
        return "mxfp4" if self.factor is None else "nvfp4"


def quantize(x: torch.Tensor, format: str = "nvfp4") -> Rows:
    """Rows [M, K] (bf16, f16, f32), any distance between them."""
    return Rows(_lib.ops().fp4_quantize(x, _format(format)), x.shape[1], format)


def swiglu_quantize(h: torch.Tensor, limit: float | None = 10.0, format: str = "nvfp4") -> Rows:
    """Limited SwiGLU (``fp8.swiglu_quantize``'s) of rows [M, 2 I] (gate columns, then up), quantized."""
    return Rows(_lib.ops().fp4_swiglu_quantize(h, limit, _format(format)), h.shape[1] // 2, format)


def quantize_weight(w: torch.Tensor, format: str = "nvfp4") -> Weights:
    """Weights [N, K] or [E, N, K] (bf16, f16, f32)."""
    return Weights(*_lib.ops().fp4_quantize_weight(w, _format(format)))


def dequantize(q: Rows | Weights, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that rows or weights stand for, rounded once (bf16 holds rows' exactly: six bits
    times a power of two)."""
    if isinstance(q, Rows):
        return _lib.ops().fp4_rows_values(q.record, q.columns, _format(q.format), dtype)
    return _lib.ops().fp4_weight_values(*q, dtype)


class PermutedRows(NamedTuple):
    """As ``permute.Permuted``, the rows quantized."""

    rows: Rows
    row_of_route: torch.Tensor
    offsets: torch.Tensor


def permute(rows: Rows, topk_ids: torch.Tensor, num_experts: int) -> PermutedRows:
    """``permute.permute`` of quantized rows: each token's record copied to its routes' rows, sorted by
    expert; a row without an expert holds zeros."""
    _lib.ops().check_records(rows.record, rows.columns, _format(rows.format))
    p = _permute(rows.record.view(torch.float8_e4m3fn), topk_ids, num_experts)  # bytes, whatever they hold
    return PermutedRows(rows._replace(record=p.rows.view(torch.uint8)), p.row_of_route, p.offsets)


def matmul(a: Rows, w: Weights, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[M, N] = quantized rows [M, K] times packed weights [N, K] transposed."""
    return _lib.ops().fp4_matmul(a.record, a.columns, _format(a.format), *w, out_dtype)


def grouped_matmul(a: Rows, offsets: torch.Tensor, w: Weights, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Rows sorted by expert (``permute``) times each expert's weights [E, N, K]: rows
    ``offsets[e] : offsets[e + 1]`` use ``w[e]``; rows before ``offsets[0]`` and from ``offsets[E]``
    on become zeros.  Offsets that fall or pass the rows are reported; those experts have no result, nor
    have later ones that go back over an earlier one's rows."""
    return _lib.ops().fp4_grouped_matmul(a.record, a.columns, _format(a.format), offsets, *w, out_dtype)


def linear(x: torch.Tensor, w: Weights, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x`` [M, K] (bf16, f16, f32) quantized to the weights' format and multiplied with packed
    weights [N, K] transposed; ``out_dtype`` defaults to x's."""
    return _lib.ops().fp4_linear(x, *w, out_dtype)
