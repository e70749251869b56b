"""8-bit floating point (E4M3) products with a scale for each block of 128.

Activations carry a scale per row and 128 columns, weights one per 128 x 128 block:

    amax = max(max |x|, 1e-30)    scale = amax / 448    q = e4m3(x * (448 / amax))

A NaN or an infinity in a block makes the whole block, and so its product's row,
NaN.  Products sum in f32.  Weights are frozen: gradients flow to activations (a
second product, of the quantized gradient with the transposed weights), never to
the packed weights.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import DTYPE_CODE, check_errors, empty, on, stream, want, want_shape  # noqa: F401

BLOCK = 128
E4M3 = torch.float8_e4m3fn
FLOATS = (torch.bfloat16, torch.float16, torch.float32)
MAX_EXPERTS = 1024


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _check_limit(limit) -> float:
    limit = float("inf") if limit is None else float(limit)
    if not limit > 0:
        raise ValueError(f"limit must be above 0 or None, got {limit}")
    return limit


def _quantize(x, width: int, swiglu: int, limit: float):
    rows, dev = x.shape[0], x.device
    q = empty(rows, width, E4M3, dev)
    scale = empty(rows, _blocks(width), torch.float32, dev)
    if rows:
        with on(dev):
            _lib.check("b200moe_fp8_quantize", _lib.lib().b200moe_fp8_quantize(
                stream(dev), x.data_ptr(), DTYPE_CODE[x.dtype], x.stride(0), rows, width, swiglu, limit,
                q.data_ptr(), scale.data_ptr()))
    return q, scale


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (bf16, f16, f32) -> (E4M3 [M, K], scale f32 [M, ceil(K / 128)])."""
    want("x", x, FLOATS, 2, rows=True)
    if x.shape[1] < 1:
        raise ValueError(f"x must have columns, got {tuple(x.shape)}")
    return _quantize(x, x.shape[1], 0, 1.0)


def swiglu_quantize(h: torch.Tensor, limit: float | None = 10.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Limited SwiGLU of rows [M, 2 I] (gate columns, then up), quantized:
    ``g / (1 + exp(-g)) * u`` with ``g = min(gate, limit)``, ``u = clamp(up, -limit, limit)``."""
    want("h", h, FLOATS, 2, rows=True)
    if h.shape[1] < 2 or h.shape[1] % 2:
        raise ValueError(f"h must have gate and up columns, got {tuple(h.shape)}")
    return _quantize(h, h.shape[1] // 2, 1, _check_limit(limit))


def swiglu_grad(h: torch.Tensor, grad: torch.Tensor, limit: float | None = 10.0) -> torch.Tensor:
    """Gradient of the SwiGLU in ``h`` [M, 2 I] for ``grad`` [M, I] of its output (the
    quantizer passes it on unchanged); zero where a bound cut the value."""
    want("h", h, FLOATS, 2, rows=True)
    want("grad", grad, (h.dtype,), 2, h.device, rows=True)
    rows, width = h.shape[0], h.shape[1] // 2
    if h.shape[1] < 2 or h.shape[1] % 2:
        raise ValueError(f"h must have gate and up columns, got {tuple(h.shape)}")
    want_shape("grad", grad, (rows, width))
    limit = _check_limit(limit)
    dev = h.device
    out = empty(rows, 2 * width, h.dtype, dev)
    if rows:
        with on(dev):
            _lib.check("b200moe_swiglu_grad", _lib.lib().b200moe_swiglu_grad(
                stream(dev), h.data_ptr(), DTYPE_CODE[h.dtype], h.stride(0), grad.data_ptr(), grad.stride(0), rows,
                width, limit, out.data_ptr()))
    return out


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights [N, K] or [E, N, K] (bf16, f16, f32) -> (E4M3 of the same shape, scale f32
    [(E,) ceil(N / 128), ceil(K / 128)])."""
    want("w", w, FLOATS, 2 if w.dim() == 2 else 3)
    if w.numel() == 0:
        raise ValueError(f"w must not be empty, got {tuple(w.shape)}")
    lead, (n, k), dev = tuple(w.shape[:-2]), w.shape[-2:], w.device
    q = torch.empty(w.shape, dtype=E4M3, device=dev)
    scale = torch.empty(lead + (_blocks(n), _blocks(k)), dtype=torch.float32, device=dev)
    with on(dev):
        _lib.check("b200moe_fp8_quantize_weight", _lib.lib().b200moe_fp8_quantize_weight(
            stream(dev), w.data_ptr(), DTYPE_CODE[w.dtype], lead[0] if lead else 1, n, k, q.data_ptr(),
            scale.data_ptr()))
    return q, scale


def transpose_weight(w: torch.Tensor, scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Packed weights [(E,) N, K] -> [(E,) K, N] with their blocks' scales: the weights
    of the product that gives the activations' gradient."""
    _check_weight(w, scale, w.dim() if isinstance(w, torch.Tensor) and w.dim() == 3 else 2, None)
    lead, (n, k), dev = tuple(w.shape[:-2]), w.shape[-2:], w.device
    out = torch.empty(lead + (k, n), dtype=E4M3, device=dev)
    out_scale = torch.empty(lead + (_blocks(k), _blocks(n)), dtype=torch.float32, device=dev)
    with on(dev):
        _lib.check("b200moe_fp8_transpose_weight", _lib.lib().b200moe_fp8_transpose_weight(
            stream(dev), w.data_ptr(), scale.data_ptr(), lead[0] if lead else 1, n, k, out.data_ptr(),
            out_scale.data_ptr()))
    return out, out_scale


def _check_weight(w, w_scale, dim: int, device) -> None:
    want("w", w, (E4M3,), dim, device)
    want("w_scale", w_scale, (torch.float32,), dim, w.device)
    n, k = w.shape[-2:]
    if w.numel() == 0:
        raise ValueError(f"w must not be empty, got {tuple(w.shape)}")
    want_shape("w_scale", w_scale, tuple(w.shape[:-2]) + (_blocks(n), _blocks(k)))


def _check_k(w, k: int) -> None:
    if w.shape[-1] != k:
        raise ValueError(f"w has {w.shape[-1]} columns, the rows {k}")
    if k % 16:
        raise ValueError(f"the product's K must be a multiple of 16, got {k}")


def _check_out(out_dtype) -> None:
    if out_dtype not in DTYPE_CODE:
        raise ValueError(f"out_dtype must be one of {'/'.join(str(d) for d in DTYPE_CODE)}, got {out_dtype}")


def _product(q, scale, offsets, w, w_scale, out_dtype):
    s, k = q.shape
    n, dev = w.shape[-2], q.device
    out = empty(s, n, out_dtype, dev)
    if s:
        with on(dev):
            _lib.check("b200moe_fp8_matmul", _lib.lib().b200moe_fp8_matmul(
                stream(dev), q.data_ptr(), scale.data_ptr(), scale.stride(0), w.data_ptr(), w_scale.data_ptr(),
                _lib.ptr(offsets), s, n, k, 1 if offsets is None else w.shape[0], out.data_ptr(),
                DTYPE_CODE[out_dtype]))
    return out


def _check_rows(q, scale) -> None:
    want("q", q, (E4M3,), 2)
    want("scale", scale, (torch.float32,), 2, q.device, rows=True)
    want_shape("scale", scale, (q.shape[0], _blocks(q.shape[1])))


def matmul(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[M, N] = quantized rows [M, K] times packed weights [N, K] transposed (K a multiple of 16)."""
    _check_rows(q, scale)
    _check_weight(w, w_scale, 2, q.device)
    _check_k(w, q.shape[1])
    _check_out(out_dtype)
    return _product(q, scale, None, w, w_scale, out_dtype)


def grouped_matmul(q: torch.Tensor, scale: torch.Tensor, offsets: torch.Tensor, w: torch.Tensor,
                   w_scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Rows sorted by expert (``permute``) times each expert's weights [E, N, K]: rows
    ``offsets[e] : offsets[e + 1]`` use ``w[e]``; rows from ``offsets[E]`` on become zeros."""
    _check_rows(q, scale)
    _check_weight(w, w_scale, 3, q.device)
    _check_k(w, q.shape[1])
    _check_out(out_dtype)
    want("offsets", offsets, (torch.int32,), 1, q.device)
    want_shape("offsets", offsets, (w.shape[0] + 1,))
    if w.shape[0] > MAX_EXPERTS or w.shape[0] * w.shape[1] > 2**31 - 257:
        raise ValueError(f"at most {MAX_EXPERTS} experts and 2^31 weight rows, got {tuple(w.shape)}")
    return _product(q, scale, offsets, w, w_scale, out_dtype)


def _linear(x, w, w_scale, out_dtype):
    (m, k), n, dev = x.shape, w.shape[0], x.device
    out = empty(m, n, out_dtype, dev)
    if m:
        # the quantized rows and their scales; few rows are quantized inside the product's kernel
        nbytes = m * (k + 4 * _blocks(k)) + 16
        if m <= 8 and x.dtype != torch.float32 and x.data_ptr() % 16 == 0 and x.stride(0) % 8 == 0:
            nbytes = _lib.lib().b200moe_fp8_linear_workspace_bytes(m, n, k)
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=dev) if nbytes else None
        with on(dev):
            _lib.check("b200moe_fp8_linear", _lib.lib().b200moe_fp8_linear(
                stream(dev), x.data_ptr(), DTYPE_CODE[x.dtype], x.stride(0), w.data_ptr(), w_scale.data_ptr(), m, n,
                k, out.data_ptr(), DTYPE_CODE[out_dtype], _lib.ptr(ws), nbytes))
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w_scale, wt, wt_scale, out_dtype):
        ctx.save_for_backward(*((w, w_scale) if wt is None else (wt, wt_scale)))
        ctx.transposed, ctx.dtype = wt is not None, x.dtype
        return _linear(x, w, w_scale, out_dtype)

    @staticmethod
    def backward(ctx, grad):
        wt, wt_scale = ctx.saved_tensors
        if not ctx.transposed:
            wt, wt_scale = transpose_weight(wt, wt_scale)
        return _linear(grad.contiguous(), wt, wt_scale, ctx.dtype), None, None, None, None, None


def linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, wt: torch.Tensor | None = None,
           wt_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x`` [M, K] (bf16, f16, f32) quantized and multiplied with packed weights [N, K]
    transposed; ``out_dtype`` defaults to x's.  Where x needs a gradient (N a multiple of
    16 then), pass ``transpose_weight``'s result as ``wt`` / ``wt_scale`` to save its
    making in each backward pass."""
    want("x", x, FLOATS, 2, rows=True)
    _check_weight(w, w_scale, 2, x.device)
    _check_k(w, x.shape[1])
    out_dtype = out_dtype or x.dtype
    _check_out(out_dtype)
    if (wt is None) != (wt_scale is None):
        raise ValueError("wt and wt_scale come together")
    if wt is not None:
        _check_weight(wt, wt_scale, 2, x.device)
        want_shape("wt", wt, (w.shape[1], w.shape[0]))
    if x.requires_grad and torch.is_grad_enabled():
        if w.shape[0] % 16:
            raise ValueError(f"the gradient's product needs N a multiple of 16, got {w.shape[0]}")
        return _Linear.apply(x, w, w_scale, wt, wt_scale, out_dtype)
    return _linear(x, w, w_scale, out_dtype)
