"""Tokens sorted by expert and back, with their gradients.

    p = permute(x, topk_ids, num_experts)          # p.rows: expert e's rows are p.offsets[e] : p.offsets[e + 1]
    y = experts(p.rows, p.offsets)
    out = unpermute(y, p.row_of_route, topk_weights)

Both take part in autograd: ``permute`` in ``x``, ``unpermute`` in ``rows`` and
``weights``.  The order is a stable sort of the T * k routes by expert id.  A route
whose id is outside ``[0, num_experts)`` (padding, an expert held elsewhere) has no
expert: its ``row_of_route`` is ``~row`` (negative), its row, after all experts'
rows, holds zeros, and it takes no part in any sum.  Sums are in f32 and in slot
order, so equal inputs give equal bits.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ops import DTYPE_CODE, check_errors, empty, on, stream, want, want_shape  # noqa: F401

FLOATS = (torch.bfloat16, torch.float16, torch.float32)
ROWS = FLOATS + (torch.float8_e4m3fn,)
MAX_EXPERTS, MAX_ROUTES, MAX_TOP_K = 1024, 1 << 26, 1024
ONE_RUN = 2048  # routes up to which the sort needs no workspace


class Permuted(NamedTuple):
    """``rows`` [T * k, H] by expert, ``scale`` [T * k, B] (None without scales),
    ``row_of_route`` int32 [T, k], ``offsets`` int32 [num_experts + 1]."""

    rows: torch.Tensor
    scale: torch.Tensor | None
    row_of_route: torch.Tensor
    offsets: torch.Tensor


def _check_routes(ids, t: int, num_experts: int, device) -> int:
    want("topk_ids", ids, (torch.int32,), 2, device)
    k = ids.shape[1]
    if ids.shape[0] != t or not 1 <= k <= MAX_TOP_K or t * k > MAX_ROUTES:
        raise ValueError(f"bad routing shape {tuple(ids.shape)} for {t} tokens")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be 1..{MAX_EXPERTS}, got {num_experts}")
    return k


def _tables(ids, num_experts: int):
    """row_of_route, offsets and the sort's workspace (None where it needs none)."""
    n, dev = ids.numel(), ids.device
    nbytes = _lib.lib().b200moe_sort_workspace_bytes(n, num_experts) if n > ONE_RUN else 0
    return (torch.empty_like(ids), torch.empty_strided((num_experts + 1,), (1,), dtype=torch.int32, device=dev),
            torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None, nbytes)


def sort_routes(topk_ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor]:
    """int32 ids [T, k] -> (row_of_route int32 [T, k], offsets int32 [num_experts + 1])."""
    want("topk_ids", topk_ids, (torch.int32,), 2)
    dev = topk_ids.device
    _check_routes(topk_ids, topk_ids.shape[0], num_experts, dev)
    row_of_route, offsets, ws, nbytes = _tables(topk_ids, num_experts)
    n = topk_ids.numel()
    if n == 0:
        return row_of_route, offsets.zero_()
    with on(dev):
        _lib.check("b200moe_sort_routes", _lib.lib().b200moe_sort_routes(
            stream(dev), topk_ids.data_ptr(), n, num_experts, row_of_route.data_ptr(), offsets.data_ptr(),
            _lib.ptr(ws), nbytes))
    return row_of_route, offsets


def _permute(x, ids, num_experts, scale):
    (t, h), k, dev = x.shape, ids.shape[1], x.device
    row_of_route, offsets, ws, nbytes = _tables(ids, num_experts)
    rows = empty(t * k, h, x.dtype, dev)
    n_scale = 0 if scale is None else scale.shape[1]
    row_scale = None if scale is None else empty(t * k, n_scale, torch.float32, dev)
    if t == 0:
        offsets.zero_()
    else:
        b = x.element_size()
        with on(dev):
            _lib.check("b200moe_permute", _lib.lib().b200moe_permute(
                stream(dev), ids.data_ptr(), num_experts, x.data_ptr(), x.stride(0) * b, h * b, _lib.ptr(scale),
                scale.stride(0) if n_scale else 0, n_scale, t, k, row_of_route.data_ptr(), offsets.data_ptr(),
                rows.data_ptr(), _lib.ptr(row_scale), _lib.ptr(ws), nbytes))
    return Permuted(rows, row_scale, row_of_route, offsets)


def _unpermute(rows, row_of_route, weights, out_dtype):
    (t, k), h, dev = row_of_route.shape, rows.shape[1], rows.device
    out = empty(t, h, out_dtype, dev)
    if t:
        with on(dev):
            _lib.check("b200moe_unpermute", _lib.lib().b200moe_unpermute(
                stream(dev), rows.data_ptr(), DTYPE_CODE[rows.dtype], row_of_route.data_ptr(), _lib.ptr(weights),
                t, k, h, out.data_ptr(), DTYPE_CODE[out_dtype]))
    return out


def unpermute_grad(grad: torch.Tensor, rows: torch.Tensor, row_of_route: torch.Tensor, weights: torch.Tensor | None,
                   need_rows: bool = True, need_weights: bool = True):
    """Gradients of ``unpermute`` in its rows and weights (None where not needed)."""
    want("rows", rows, FLOATS, 2)
    dev = rows.device
    want("grad", grad, (rows.dtype, torch.float32), 2, dev, rows=True)
    _check_row_of_route(row_of_route, rows, weights)
    (t, k), h = row_of_route.shape, rows.shape[1]
    want_shape("grad", grad, (t, h))
    need_weights = need_weights and weights is not None
    grad_rows = torch.empty_like(rows) if need_rows else None
    grad_weights = torch.empty_like(weights) if need_weights else None
    if t and (need_rows or need_weights):
        with on(dev):
            _lib.check("b200moe_unpermute_grad", _lib.lib().b200moe_unpermute_grad(
                stream(dev), grad.data_ptr(), DTYPE_CODE[grad.dtype], grad.stride(0), rows.data_ptr(),
                DTYPE_CODE[rows.dtype], row_of_route.data_ptr(), _lib.ptr(weights), t, k, h, _lib.ptr(grad_rows),
                _lib.ptr(grad_weights)))
    return grad_rows, grad_weights


def _check_row_of_route(row_of_route, rows, weights):
    dev = rows.device
    want("row_of_route", row_of_route, (torch.int32,), 2, dev)
    t, k = row_of_route.shape
    if rows.shape[0] != t * k or rows.shape[1] < 1 or not 1 <= k <= MAX_TOP_K or t * k > MAX_ROUTES:
        raise ValueError(f"rows {tuple(rows.shape)} do not fit the routes {tuple(row_of_route.shape)}")
    if weights is not None:
        want("weights", weights, (torch.float32,), 2, dev)
        want_shape("weights", weights, (t, k))


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts):
        p = _permute(x, ids, num_experts, None)
        ctx.save_for_backward(p.row_of_route)
        ctx.mark_non_differentiable(p.row_of_route, p.offsets)
        ctx.set_materialize_grads(False)
        return p.rows, p.row_of_route, p.offsets

    @staticmethod
    def backward(ctx, grad, *_):
        if grad is None:
            return None, None, None
        row_of_route, = ctx.saved_tensors
        return _unpermute(grad.contiguous(), row_of_route, None, grad.dtype), None, None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, row_of_route, weights, out_dtype):
        ctx.save_for_backward(rows, row_of_route, weights)
        return _unpermute(rows, row_of_route, weights, out_dtype)

    @staticmethod
    def backward(ctx, grad):
        rows, row_of_route, weights = ctx.saved_tensors
        if grad.stride(-1) != 1 or grad.stride(0) < grad.shape[1]:
            grad = grad.contiguous()
        grad_rows, grad_weights = unpermute_grad(grad, rows, row_of_route, weights, ctx.needs_input_grad[0],
                                                 ctx.needs_input_grad[2])
        return grad_rows, None, grad_weights, None


def permute(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int, scale: torch.Tensor | None = None) -> Permuted:
    """Copy each token's row of ``x`` [T, H] (bf16, f16, f32, or E4M3 with its ``scale``
    f32 [T, B]) to its routes' rows, sorted by expert (``topk_ids`` int32 [T, k])."""
    want("x", x, ROWS, 2, rows=True)
    t, h = x.shape
    if h < 1:
        raise ValueError(f"x must have columns, got {tuple(x.shape)}")
    _check_routes(topk_ids, t, num_experts, x.device)
    if scale is not None:
        want("scale", scale, (torch.float32,), 2, x.device, rows=True)
        if scale.shape[0] != t:
            raise ValueError(f"scale must have {t} rows, got {tuple(scale.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        if scale is not None:
            raise ValueError("rows with scales are quantized: permute them without gradient")
        rows, row_of_route, offsets = _Permute.apply(x, topk_ids, num_experts)
        return Permuted(rows, None, row_of_route, offsets)
    return _permute(x, topk_ids, num_experts, scale)


def unpermute(rows: torch.Tensor, row_of_route: torch.Tensor, weights: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``out[t] = sum_s weights[t, s] * rows[row_of_route[t, s]]`` over the routes that
    have an expert (``weights`` f32 [T, k], None: ones); ``out_dtype``: the rows' or f32."""
    want("rows", rows, FLOATS, 2)
    _check_row_of_route(row_of_route, rows, weights)
    out_dtype = out_dtype or rows.dtype
    if out_dtype not in (rows.dtype, torch.float32):
        raise ValueError(f"out_dtype must be {rows.dtype} or torch.float32, got {out_dtype}")
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        return _Unpermute.apply(rows, row_of_route, weights, out_dtype)
    return _unpermute(rows, row_of_route, weights, out_dtype)
