"""A decoder's expert block on 4-bit experts: the norm's gain learns in front of FP8 experts, then the block serves in 4 bits.

    python examples/fp4_block.py [--tokens 512 --hidden 1024 --inter 512 --experts 32 --top-k 4 --steps 20]

Training runs the residual's addition and norm with their gradients and FP8 experts behind them; serving runs the same
norm with its rows quantized in one pass (the router reads them before that), 4-bit experts from those rows, and one
token at a time.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))


def route(y, router, top_k):
    """Softmax top-k with renormalised weights: int32 ids and fp32 weights."""
    top, ids = (y.float() @ router.t()).topk(top_k, dim=1)
    return ids.to(torch.int32), top.softmax(-1).contiguous()


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("tokens", 512), ("hidden", 1024), ("inter", 512), ("experts", 32), ("top-k", 4),
                          ("steps", 20)):
        ap.add_argument("--" + name, type=int, default=default)
    a = ap.parse_args(argv)
    from __graft_entry__ import load_package

    load_package()
    from b200moe import norm
    from b200moe.experts import Fp4Experts, Fp8Experts

    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w13, w2 = rand(a.experts, 2 * a.inter, a.hidden) * a.hidden**-0.5, rand(a.experts, a.hidden, a.inter) * a.inter**-0.5
    router = rand(a.experts, a.hidden) * a.hidden**-0.5
    x, stream = rand(a.tokens, a.hidden).bfloat16(), rand(a.tokens, a.hidden)  # the residual stream stays in f32

    layer = Fp8Experts.from_weights(w13, w2, trainable=True)
    target = 1 + 0.2 * rand(a.hidden)
    gain = torch.ones(a.hidden, device="cuda", requires_grad=True)
    opt = torch.optim.Adam([gain], lr=2e-2)
    with torch.no_grad():
        y, _ = norm.rms_norm(x, target, stream)
        want = layer(y, *route(y, router, a.top_k)).float()
    losses, grad = [], 0.0
    for _ in range(a.steps):
        opt.zero_grad()
        y, total = norm.rms_norm(x, gain, stream)
        loss = (layer(y, *route(y.detach(), router, a.top_k)).float() - want).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        grad = gain.grad.abs().mean()
    losses = torch.stack(losses).tolist()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")

    served = {}
    with torch.no_grad():
        want = layer(y := norm.rms_norm(x, gain, stream).y, *route(y, router, a.top_k)).float()
        for fmt in ("nvfp4", "mxfp4"):
            experts = Fp4Experts.from_weights(w13, w2, fmt)

            def block(rows, s):
                n = norm.rms_norm_quantize(rows, gain, s, format=fmt, keep=True)
                return experts(n.rows, *route(n.y, router, a.top_k))

            out = block(x, stream)
            single = torch.cat([block(x[i: i + 1], stream[i: i + 1]) for i in range(8)])
            served[fmt] = float((out.float() - want).norm() / want.norm())
            off = float((single.float() - out[:8].float()).norm() / out[:8].float().norm())
            print(f"{fmt}: {served[fmt]:.3f} relative to the FP8 experts; single tokens against the batch {off:.1e}")
    return {"first": losses[0], "last": losses[-1], "gain_gradient": float(grad), **served}


if __name__ == "__main__":
    main()
