"""FP8 routed experts: the operators of ``permute`` and ``fp8`` run together.

``Fp8Experts`` holds frozen E4M3 experts (a scale per 128 x 128 block) and computes
the weighted sum of each token's top-k experts, for serving and, through autograd,
with the gradients of the tokens and the router weights.  The counterpart, for
experts kept in FP8, of ``moe.B200NativeMoe``; its SwiGLU and its routing contract
(int32 ids, fp32 weights) are the same.
"""

from __future__ import annotations

import torch

from . import _lib, fp8
from .permute import permute, unpermute, unpermute_grad

SWIGLU_LIMIT = 10.0


class Fp8Experts:
    """``w13`` E4M3 [E, 2 I, H] (gate rows, then up rows) and ``w2`` [E, H, I] with their
    scales (``fp8.quantize_weight``); H and I multiples of 16.  ``trainable`` also keeps
    the transposed weights, which the tokens' gradient needs (the router weights' does not)."""

    def __init__(self, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor, *,
                 swiglu_limit: float | None = SWIGLU_LIMIT, trainable: bool = False):
        _lib.ops().check_weight("w13", w13, w13_scale)
        _lib.ops().check_weight("w2", w2, w2_scale)
        e, i2, h = w13.shape
        if w2.shape != (e, h, i2 // 2) or i2 % 32 or h % 16 or e > 1024 or w2.device != w13.device:
            raise ValueError("w13 [E, 2 I, H] and w2 [E, H, I] need H and I multiples of 16, E at most 1024 and one "
                             f"device, got {tuple(w13.shape)} and {tuple(w2.shape)}")
        self.num_experts, self.hidden, self.inter = e, h, i2 // 2
        self.w13, self.w13_scale, self.w2, self.w2_scale = w13, w13_scale, w2, w2_scale
        self.swiglu_limit = swiglu_limit
        self.w13_t = self.w13_t_scale = self.w2_t = self.w2_t_scale = None
        if trainable:
            self.w13_t, self.w13_t_scale = fp8.transpose_weight(w13, w13_scale)
            self.w2_t, self.w2_t_scale = fp8.transpose_weight(w2, w2_scale)

    @classmethod
    def from_weights(cls, w13: torch.Tensor, w2: torch.Tensor, **kw) -> "Fp8Experts":
        """Quantizes full-precision weights [E, 2 I, H] and [E, H, I]."""
        return cls(*fp8.quantize_weight(w13), *fp8.quantize_weight(w2), **kw)

    def _products(self, x, topk_ids):
        """(h [S, 2 I], y [S, H], row_of_route, offsets) of the sorted routes."""
        q, scale = fp8.quantize(x)  # once per token, not once per route
        p = permute(q, topk_ids, self.num_experts, scale=scale)
        h = fp8.grouped_matmul(p.rows, p.scale, p.offsets, self.w13, self.w13_scale, x.dtype)
        a, a_scale = fp8.swiglu_quantize(h, self.swiglu_limit)
        y = fp8.grouped_matmul(a, a_scale, p.offsets, self.w2, self.w2_scale, x.dtype)
        return h, y, p.row_of_route, p.offsets

    def forward(self, x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor) -> torch.Tensor:
        """x [T, H] (bf16 or f16), int32 ids and fp32 weights [T, k] -> [T, H] in x's dtype.
        An id outside [0, E) contributes nothing."""
        if x.dtype not in (torch.bfloat16, torch.float16) or x.dim() != 2 or x.shape[1] != self.hidden or \
                x.device != self.w13.device:
            raise ValueError(f"x must be fp16 or bf16 [T, {self.hidden}] on {self.w13.device}, got {x.dtype} "
                             f"{tuple(x.shape)} on {x.device}")
        if topk_weights.shape != topk_ids.shape:
            raise ValueError(f"bad routing shape {tuple(topk_ids.shape)} with weights {tuple(topk_weights.shape)}")
        if torch.is_grad_enabled() and (x.requires_grad or topk_weights.requires_grad):
            if x.requires_grad and self.w13_t is None:
                raise ValueError("the tokens' gradient needs trainable=True (the transposed weights)")
            return _Experts.apply(x, topk_weights, topk_ids, self)
        _, y, row_of_route, _ = self._products(x, topk_ids)
        return unpermute(y, row_of_route, topk_weights)

    __call__ = forward


class _Experts(torch.autograd.Function):
    """The quantizers pass gradients on unchanged; the gradients that enter the two
    products are quantized like their activations."""

    @staticmethod
    def forward(ctx, x, topk_weights, topk_ids, experts):
        h, y, row_of_route, offsets = experts._products(x, topk_ids)
        ctx.save_for_backward(h, y, row_of_route, offsets, topk_weights)
        ctx.experts = experts
        return unpermute(y, row_of_route, topk_weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        h, y, row_of_route, offsets, w = ctx.saved_tensors
        m = ctx.experts
        need_x, need_w = ctx.needs_input_grad[:2]
        gy, gw = unpermute_grad(grad.contiguous(), y, row_of_route, w, need_x, need_w)
        if not need_x:
            return None, gw, None, None
        q, scale = fp8.quantize(gy)
        ga = fp8.grouped_matmul(q, scale, offsets, m.w2_t, m.w2_t_scale, h.dtype)
        q, scale = fp8.quantize(fp8.swiglu_grad(h, ga, m.swiglu_limit))
        gx = fp8.grouped_matmul(q, scale, offsets, m.w13_t, m.w13_t_scale, h.dtype)
        return unpermute(gx, row_of_route), gw, None, None
