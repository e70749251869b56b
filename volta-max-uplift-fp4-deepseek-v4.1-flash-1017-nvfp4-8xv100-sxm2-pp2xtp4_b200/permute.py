"""Tokens sorted by expert and back, with their gradients.

    p = permute(x, topk_ids, num_experts)          # p.rows: expert e's rows are p.offsets[e] : p.offsets[e + 1]
    y = experts(p.rows, p.offsets)
    out = unpermute(y, p.row_of_route, topk_weights)

Both take part in autograd: ``permute`` in ``x``, ``unpermute`` in ``rows`` and
``weights``.  The order is a stable sort of the T * k routes by expert id.  A route
whose id is outside ``[0, num_experts)`` (padding, an expert held elsewhere) has no
expert: its ``row_of_route`` is ``~row`` (negative), its row, after all experts'
rows, holds zeros, and it takes no part in any sum.  Sums are in f32 and in slot
order, so equal inputs give equal bits.  Arguments that do not fit raise
``ValueError``; a ``row_of_route`` entry out of range is left out and reported by
``check_errors``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ops import check_errors  # noqa: F401


class Permuted(NamedTuple):
    """``rows`` [T * k, H] by expert, ``scale`` [T * k, B] (None without scales),
    ``row_of_route`` int32 [T, k], ``offsets`` int32 [num_experts + 1]."""

    rows: torch.Tensor
    scale: torch.Tensor | None
    row_of_route: torch.Tensor
    offsets: torch.Tensor


def sort_routes(topk_ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor]:
    """int32 ids [T, k] -> (row_of_route int32 [T, k], offsets int32 [num_experts + 1]).
    At most 1024 experts and 2^26 routes.  Every 2048 routes read the counts of all the
    others, so the time grows with the square of the routes: 13 us at 131,072 of them
    (384 experts), 88 us at 2^20, 3.7 ms at 2^23."""
    return _lib.ops().sort_routes(topk_ids, num_experts)


def permute(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int, scale: torch.Tensor | None = None) -> Permuted:
    """Copy each token's row of ``x`` [T, H] (bf16, f16, f32, or E4M3 with its ``scale``
    f32 [T, B]) to its routes' rows, sorted by expert (``topk_ids`` int32 [T, k]).
    E4M3 rows and rows with scales have no gradient: where ``x`` requires one they are refused."""
    return Permuted(*_lib.ops().permute(x, topk_ids, num_experts, scale))


def unpermute(rows: torch.Tensor, row_of_route: torch.Tensor, weights: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``out[t] = sum_s weights[t, s] * rows[row_of_route[t, s]]`` over the routes that
    have an expert (``weights`` f32 [T, k], None: ones); ``out_dtype``: the rows' or f32.
    ``row_of_route`` is ``permute``'s or another map of the same form: the gradients
    need every row named exactly once, also those of dropped routes (``~row``, not any
    negative number), since each row's gradient is written by the route that names it."""
    return _lib.ops().unpermute(rows, row_of_route, weights, out_dtype)


def unpermute_grad(grad: torch.Tensor, rows: torch.Tensor, row_of_route: torch.Tensor, weights: torch.Tensor | None,
                   need_rows: bool = True, need_weights: bool = True):
    """Gradients of ``unpermute`` in its rows and weights (None where not needed)."""
    return _lib.ops().unpermute_grad(grad, rows, row_of_route, weights, need_rows, need_weights)
