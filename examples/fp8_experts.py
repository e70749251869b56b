"""FP8 routed experts: a router learns on frozen experts, then the layer serves single tokens.

    python examples/fp8_experts.py [--tokens 512 --hidden 1024 --inter 512 --experts 32 --top-k 4 --steps 40]

The data is random and the target comes from a teacher router, so the loss falls as the learned router comes to
choose and weigh the experts as the teacher does. The operators it runs: the row quantizer, the sort by expert with its
copies, the grouped FP8 products, the SwiGLU quantizer, the weighted return and all their gradients.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))


def route(x, router, top_k):
    """Softmax top-k with renormalised weights: int32 ids and the fp32 weights that carry the gradient."""
    logits = x.float() @ router.t()
    top, ids = logits.topk(top_k, dim=1)
    return ids.to(torch.int32), top.softmax(-1).contiguous()


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("tokens", 512), ("hidden", 1024), ("inter", 512), ("experts", 32), ("top-k", 4),
                          ("steps", 40)):
        ap.add_argument("--" + name, type=int, default=default)
    a = ap.parse_args(argv)
    from __graft_entry__ import load_package

    load_package()
    from b200moe.experts import Fp8Experts

    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    layer = Fp8Experts.from_weights(rand(a.experts, 2 * a.inter, a.hidden) * a.hidden**-0.5,
                                    rand(a.experts, a.hidden, a.inter) * a.inter**-0.5, trainable=True)
    x = rand(a.tokens, a.hidden).bfloat16()
    teacher = rand(a.experts, a.hidden) * a.hidden**-0.5
    with torch.no_grad():
        target = layer(x, *route(x, teacher, a.top_k)).float()
    router = (teacher + 0.5 * rand(a.experts, a.hidden) * a.hidden**-0.5).requires_grad_()
    opt = torch.optim.Adam([router], lr=2e-3)
    losses = []
    for _ in range(a.steps):
        opt.zero_grad()
        loss = (layer(x, *route(x, router, a.top_k)).float() - target).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    with torch.no_grad():  # serving: one token at a time gives the batch's rows
        batch = layer(x[:8], *route(x[:8], router, a.top_k))
        single = torch.cat([layer(x[i: i + 1], *route(x[i: i + 1], router, a.top_k)) for i in range(8)])
    off = float((batch.float() - single.float()).norm() / batch.float().norm())
    print(f"single tokens against the batch: {off:.1e} relative")
    return {"first": losses[0], "last": losses[-1], "single": off}


if __name__ == "__main__":
    main()
