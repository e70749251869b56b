"""Cases that time and check the operators of the FP8 expert path against plain torch forms.

The operators are the public calls of the package's ``permute`` and ``fp8`` modules:

- ``permute``   tokens copied into rows sorted by expert (``permute.permute``), and its gradient;
- ``unpermute`` expert rows back to token order, weighted and summed (``permute.unpermute``), and its gradients;
- ``quantize``  rows to 8-bit floating point (E4M3) with one scale per 128 columns, after a limited SwiGLU or
  none (``fp8.quantize``, ``fp8.swiglu_quantize``), and the SwiGLU's gradient (``fp8.swiglu_grad``);
- ``linear``    y = x . W^T with E4M3 operands, x quantized in the call (``fp8.linear``), and the gradient of x;
- ``grouped``   the same product of rows sorted by expert with each expert's own weights (``fp8.grouped_matmul``).

With ``own`` false, ``run`` computes the plain form; with ``own`` true it makes the package's calls.
"""

import math
import random

import torch

own = False

BLOCK = 128  # columns (and, for weights, rows) that share one scale
E4M3_MAX = 448.0
AMAX_FLOOR = 1e-30
LIMIT = 10.0  # the framework's SwiGLU bound
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one generated token's quantized row and its scales sent to its eight experts: launch latency
        {"name": "permute_token", "op": "permute", "tokens": 1, "hidden": 4096, "experts": 384, "top_k": 8,
         "dtype": "fp8", "skew": 0.0, "drop": 0.0, "train": False},
        # a ragged fine-tuning batch of the smaller layer, with padding routes that have no expert
        {"name": "permute_train_ragged", "op": "permute", "tokens": 1013, "hidden": 2048, "experts": 64, "top_k": 6,
         "dtype": "f16", "skew": 1.1, "drop": 0.1, "train": True},
        # the longest prompt of the prefill layer, forward and backward
        {"name": "permute_train_16k", "op": "permute", "tokens": 16384, "hidden": 4096, "experts": 384, "top_k": 8,
         "dtype": "bf16", "skew": 0.0, "drop": 0.0, "train": True},
        # the weighted return of the largest decode batch
        {"name": "unpermute_batch64", "op": "unpermute", "tokens": 64, "hidden": 4096, "experts": 384, "top_k": 8,
         "dtype": "bf16", "skew": 0.0, "drop": 0.0, "train": False},
        # the weighted return of a training batch with the gradients of rows and router weights
        {"name": "unpermute_train_4k", "op": "unpermute", "tokens": 4096, "hidden": 4096, "experts": 384, "top_k": 8,
         "dtype": "bf16", "skew": 1.1, "drop": 0.05, "train": True},
        # SwiGLU rows of a decode batch (32 tokens, 8 experts each) quantized for the down projection
        {"name": "swiglu_decode", "op": "quantize", "rows": 256, "width": 2048, "act": "swiglu", "dtype": "bf16",
         "train": False},
        # the same of a training batch at the smaller layer's width (11 blocks of 128), with the gradient
        {"name": "swiglu_train_48k", "op": "quantize", "rows": 49152, "width": 1408, "act": "swiglu",
         "dtype": "bf16", "train": True},
        # one token through a dense projection: weights streamed once
        {"name": "linear_token", "op": "linear", "tokens": 1, "n": 4096, "k": 4096, "dtype": "bf16", "train": False},
        # a ragged batch through the smaller layer's projection, with the gradient of x
        {"name": "linear_train_ragged", "op": "linear", "tokens": 333, "n": 2816, "k": 2048, "dtype": "bf16",
         "train": True},
        # a long prompt through the dense projection: tensor-bound
        {"name": "linear_8k", "op": "linear", "tokens": 8192, "n": 4096, "k": 4096, "dtype": "bf16", "train": False},
        # 32 decoding tokens over 384 experts: about 190 experts' weights streamed for one or two rows each
        {"name": "grouped_decode", "op": "grouped", "tokens": 32, "experts": 384, "top_k": 8, "n": 4096, "k": 4096,
         "skew": 0.0, "drop": 0.0},
        # a long prompt over the smaller layer's 64 experts, unevenly loaded: tensor-bound
        {"name": "grouped_prefill", "op": "grouped", "tokens": 6000, "experts": 64, "top_k": 6, "n": 2816, "k": 2048,
         "skew": 0.5, "drop": 0.0},
    ]


def _log(rng, lo, hi):
    """Spread over the logarithm; odd above 64, where nothing else would leave a ragged last tile."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n if n <= 64 else min(n | 1, hi)


def _sixteens(rng, lo, hi):
    """A width of whole 16-byte pieces of E4M3 values, mostly no multiple of 128."""
    return 16 * (rng.randint(lo // 16, hi // 16) | 1)


def draw(rng):
    op = rng.choice(["permute", "unpermute", "quantize", "linear", "grouped"])
    if op in ("permute", "unpermute"):
        experts, top_k = rng.choice([(384, 8), (64, 6), (rng.randint(8, 500), rng.randint(1, 8))])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"] + (["fp8"] if op == "permute" else []))
        # odd widths too; an FP8 row keeps whole 16-byte pieces, as its matrix product wants it
        hidden = rng.choice([4096, 2048, _sixteens(rng, 256, 4000), rng.randint(256, 4000) | 1])
        if dtype == "fp8" and hidden % 16:
            hidden = _sixteens(rng, 256, 4000)
        return {"op": op, "tokens": _log(rng, 1, 8192 if dtype == "f32" else 16384), "hidden": hidden,
                "experts": experts, "top_k": top_k, "dtype": dtype, "skew": rng.choice([0.0, 0.5, 1.1]),
                "drop": rng.choice([0.0, 0.0, 0.1, 0.5]), "train": dtype != "fp8" and rng.random() < 0.5}
    if op == "quantize":
        act = rng.choice(["swiglu", "none"])
        return {"op": op, "rows": _log(rng, 1, 49152), "width": rng.choice([1408, 2048, 4096, rng.randint(1, 4000) | 1])
                if act == "none" else rng.choice([1408, rng.randint(1, 1400) | 1]), "act": act,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "train": act == "swiglu" and rng.random() < 0.5}
    n, k = rng.choice([(4096, 4096), (4096, 2048), (2816, 2048), (2048, 1408),
                       (rng.randint(64, 4000) | 1, _sixteens(rng, 128, 4000))])
    if op == "linear":
        train = rng.random() < 0.3
        if train and n % 16:  # the gradient contracts over n: whole 16-byte pieces of the transposed weights
            n = _sixteens(rng, 64, 4000)
        return {"op": op, "tokens": _log(rng, 1, 4096 if train else 8192), "n": n, "k": k,
                "dtype": rng.choice(["bf16", "bf16", "f16"]), "train": train}
    experts, top_k = rng.choice([(64, 6), (384, 8), (rng.randint(4, 128), rng.randint(1, 4))])
    most = 6000 * 6 * 2816 * 2048 // (n * k * top_k)  # no more work than the largest listed case
    return {"op": op, "tokens": _log(rng, 1, max(2, min(6000, most))), "experts": experts, "top_k": top_k, "n": n,
            "k": k, "skew": rng.choice([0.0, 0.5]), "drop": rng.choice([0.0, 0.0, 0.1])}


# ------------------------------------------------------------------ inputs
def _routing(g, case):
    """Expert ids int32 [T, k]: the k largest of normal logits, with a Zipf bias of exponent `skew` on the experts'
    popularity; a share `drop` of the routes has no expert (-1), as padding and experts held elsewhere do."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn(t, e, generator=g, device="cuda")
    rank = torch.randperm(e, generator=g, device="cuda").float() + 1
    logits = logits - case["skew"] * rank.log()
    ids = logits.topk(k, dim=1).indices.to(torch.int32)
    if case["drop"] > 0:
        gone = torch.rand(t, k, generator=g, device="cuda") < case["drop"]
        ids = torch.where(gone, torch.full_like(ids, -1), ids)
    return ids.contiguous()


def _activations(g, rows, width, dtype):
    """Normal values with a few wide columns, as hidden states have them."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    wide = torch.rand(width, generator=g, device="cuda") < 0.01
    return (x * torch.where(wide, 12.0, 1.0)).to(dtype)


def _weights(g, lead, n, k):
    """E4M3 weights [*lead, n, k] of N(0, 0.02) with one scale per block of 128 x 128."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    count = math.prod(lead)
    q = torch.empty((count, n, k), dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty((count, nb, kb), device="cuda")
    for i in range(count):
        w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
        w[:n, :k] = 0.02 * torch.randn(n, k, generator=g, device="cuda")
        blocks = w.view(nb, BLOCK, kb, BLOCK)
        scale[i] = blocks.abs().amax(dim=(1, 3)).clamp_min(AMAX_FLOOR) / E4M3_MAX
        w = (blocks / scale[i][:, None, :, None]).view(nb * BLOCK, kb * BLOCK)
        q[i] = w[:n, :k].clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(*lead, n, k), scale.view(*lead, nb, kb)


def _sorted_routes(ids, experts):
    """(order, offsets): routes sorted by expert, ties by route, those without an expert last; where each expert's
    rows begin."""
    key = ids.reshape(-1).long()
    key = torch.where((key < 0) | (key >= experts), experts, key)
    order = torch.argsort(key, stable=True)
    offsets = torch.searchsorted(key[order], torch.arange(experts + 1, device=key.device)).to(torch.int32)
    return order, offsets


def _row_of_route(order, offsets, shape):
    """Row of each route; a route without an expert has ~row, the row of zeros kept for it."""
    at = torch.arange(order.numel(), device=order.device)
    row = torch.empty_like(order)
    row[order] = torch.where(at < offsets[-1], at, ~at)
    return row.to(torch.int32).view(shape)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op in ("permute", "unpermute"):
        t, k, h = case["tokens"], case["top_k"], case["hidden"]
        dt = DTYPES[case["dtype"]]
        s["ids"] = _routing(g, case)
        if op == "permute":
            x = _activations(g, t, h, torch.float32)
            if case["dtype"] == "fp8":
                s["x"], s["scale"] = _quantize(x)
            else:
                s["x"] = x.to(dt)
            if case["train"]:
                s["grad"] = torch.randn(t * k, h, generator=g, device="cuda").to(dt)
        else:
            order, offsets = _sorted_routes(s["ids"], case["experts"])
            s["row_of_route"] = _row_of_route(order, offsets, (t, k))
            s["rows"] = torch.randn(t * k, h, generator=g, device="cuda").to(dt)
            s["weights"] = torch.rand(t, k, generator=g, device="cuda").softmax(-1)
            if case["train"]:
                s["grad"] = torch.randn(t, h, generator=g, device="cuda").to(dt)
    elif op == "quantize":
        dt, width = DTYPES[case["dtype"]], case["width"]
        s["x"] = _activations(g, case["rows"], 2 * width if case["act"] == "swiglu" else width, dt)
        if case["train"]:
            s["grad"] = torch.randn(case["rows"], width, generator=g, device="cuda").to(dt)
    elif op == "linear":
        s["x"] = _activations(g, case["tokens"], case["k"], DTYPES[case["dtype"]])
        s["w"], s["w_scale"] = _weights(g, (), case["n"], case["k"])
        if case["train"]:  # a program that trains keeps the transposed weights too
            s["wt"], s["wt_scale"] = s["w"].view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn), \
                s["w_scale"].t().contiguous()
            s["grad"] = _activations(g, case["tokens"], case["n"], DTYPES[case["dtype"]])
    else:
        s["ids"] = _routing(g, case)
        order, s["offsets"] = _sorted_routes(s["ids"], case["experts"])
        s["q"], s["scale"] = _quantize(_activations(g, order.numel(), case["k"], torch.float32))
        s["w"], s["w_scale"] = _weights(g, (case["experts"],), case["n"], case["k"])
        # the plain form's padded batch: most rows of one expert
        s["most"] = max(1, int((s["offsets"][1:] - s["offsets"][:-1]).max()))
    return s


# ------------------------------------------------------------- plain forms
def _blocks(x):
    """[rows, width] -> [rows, blocks, 128], zeros after the last column."""
    rows, width = x.shape
    kb = -(-width // BLOCK)
    if kb * BLOCK != width:
        x = torch.cat([x, x.new_zeros(rows, kb * BLOCK - width)], dim=1)
    return x.reshape(rows, kb, BLOCK)


def _quantize(x):
    """f32 [rows, width] -> E4M3 values and scales amax / 448 [rows, blocks]."""
    b = _blocks(x)
    amax = b.abs().amax(-1).clamp_min(AMAX_FLOOR)
    top = torch.full_like(amax, E4M3_MAX)  # a quotient with a plain number would be a product with its reciprocal
    q = (b * (top / amax)[..., None]).to(torch.float8_e4m3fn)
    return q.view(x.shape[0], -1)[:, : x.shape[1]].contiguous(), amax / top


def _dequantize(q, scale):
    wide = scale.repeat_interleave(BLOCK, dim=-1)[..., : q.shape[-1]]
    return q.float() * wide


def _dequantize_weights(w, scale):
    return _dequantize(w, scale.repeat_interleave(BLOCK, dim=-2)[..., : w.shape[-2], :])


def _plain_permute(s):
    case, ids, x = s["case"], s["ids"], s["x"]
    t, k = ids.shape
    order, offsets = _sorted_routes(ids, case["experts"])
    out = {"row_of_route": _row_of_route(order, offsets, (t, k)), "offsets": offsets}
    held = (torch.arange(t * k, device=x.device) < offsets[-1])[:, None]
    if case["dtype"] == "fp8":
        rows = torch.where(held, x.view(torch.uint8)[order // k], 0).to(torch.uint8)
        out["rows"] = rows.view(torch.float8_e4m3fn)
        out["scale"] = torch.where(held, s["scale"][order // k], 0.0)
    else:
        out["rows"] = torch.where(held, x[order // k], torch.zeros((), dtype=x.dtype, device=x.device))
    if case["train"]:
        row = out["row_of_route"].long()
        back = s["grad"].float()[row.clamp_min(0)]
        out["grad_x"] = torch.where((row >= 0)[..., None], back, 0.0).sum(1).to(x.dtype)
    return out


def _plain_unpermute(s):
    row, rows, w = s["row_of_route"].long(), s["rows"], s["weights"]
    held = (row >= 0)[..., None]
    y = torch.where(held, rows.float()[row.clamp_min(0)], 0.0)
    out = {"out": (w[..., None] * y).sum(1).to(rows.dtype)}
    if s["case"]["train"]:
        g = s["grad"].float()
        back = torch.where(held, w[..., None] * g[:, None], 0.0)
        grad_rows = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
        grad_rows[torch.where(row < 0, ~row, row).view(-1)] = back.view(rows.shape).to(rows.dtype)
        out["grad_rows"] = grad_rows
        out["grad_weights"] = (g[:, None] * y).sum(-1)
    return out


def _plain_quantize(s):
    case, x = s["case"], s["x"].float()
    if case["act"] == "none":
        q, scale = _quantize(x)
        return {"q": q, "scale": scale}
    gate, up = x[:, : case["width"]], x[:, case["width"]:]
    g, u = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
    e = torch.exp(-g)
    q, scale = _quantize(g / (1 + e) * u)
    out = {"q": q, "scale": scale}
    if case["train"]:
        d = s["grad"].float()
        sig = 1 / (1 + e)
        dg = torch.where(gate > LIMIT, 0.0, d * u * (sig * (1 + g * (1 - sig))))
        du = torch.where(up.abs() > LIMIT, 0.0, d * (g * sig))
        out["grad_x"] = torch.cat([dg, du], dim=1).to(s["x"].dtype)
    return out


def _plain_linear(s):
    x = s["x"]
    w = _dequantize_weights(s["w"], s["w_scale"])
    out = {"y": (_dequantize(*_quantize(x.float())) @ w.t()).to(x.dtype)}
    if s["case"]["train"]:
        out["grad_x"] = (_dequantize(*_quantize(s["grad"].float())) @ w).to(x.dtype)
    return out


def _plain_grouped(s):
    case, off, q = s["case"], s["offsets"].long(), s["q"]
    at = torch.arange(q.shape[0], device=q.device)
    expert = torch.searchsorted(off[1:].contiguous(), at, right=True).clamp_max(case["experts"] - 1)
    held = (at < off[-1])[:, None]
    place = (at - off[expert]).clamp_max(s["most"])  # rows without an expert go to a place of their own
    x = q.new_zeros((case["experts"], s["most"] + 1, case["k"]), dtype=torch.float32)
    x[expert, place] = torch.where(held, _dequantize(q, s["scale"]), 0.0)
    y = x[:, : s["most"]] @ _dequantize_weights(s["w"], s["w_scale"]).transpose(1, 2)
    y = torch.where(held, y[expert, place.clamp_max(s["most"] - 1)], 0.0)
    return {"y": y.to(torch.bfloat16)}


PLAIN = {"permute": _plain_permute, "unpermute": _plain_unpermute, "quantize": _plain_quantize,
         "linear": _plain_linear, "grouped": _plain_grouped}


# ---------------------------------------------------------- the package's calls
def _package():
    from __graft_entry__ import load_package

    load_package()
    from b200moe import fp8, permute

    return permute, fp8


def _own_permute(s):
    permute, _ = _package()
    case, x = s["case"], s["x"]
    if not case["train"]:
        p = permute.permute(x, s["ids"], case["experts"], scale=s.get("scale"))
        out = {"row_of_route": p.row_of_route, "offsets": p.offsets, "rows": p.rows}
        return out if p.scale is None else {**out, "scale": p.scale}
    x = x.detach().requires_grad_()
    p = permute.permute(x, s["ids"], case["experts"])
    grad_x, = torch.autograd.grad(p.rows, x, s["grad"])
    return {"row_of_route": p.row_of_route, "offsets": p.offsets, "rows": p.rows, "grad_x": grad_x}


def _own_unpermute(s):
    permute, _ = _package()
    if not s["case"]["train"]:
        return {"out": permute.unpermute(s["rows"], s["row_of_route"], s["weights"])}
    rows, w = s["rows"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
    out = permute.unpermute(rows, s["row_of_route"], w)
    grad_rows, grad_w = torch.autograd.grad(out, (rows, w), s["grad"])
    return {"out": out, "grad_rows": grad_rows, "grad_weights": grad_w}


def _own_quantize(s):
    _, fp8 = _package()
    if s["case"]["act"] == "none":
        q, scale = fp8.quantize(s["x"])
        return {"q": q, "scale": scale}
    q, scale = fp8.swiglu_quantize(s["x"], limit=LIMIT)
    out = {"q": q, "scale": scale}
    if s["case"]["train"]:
        out["grad_x"] = fp8.swiglu_grad(s["x"], s["grad"], limit=LIMIT)
    return out


def _own_linear(s):
    _, fp8 = _package()
    if not s["case"]["train"]:
        return {"y": fp8.linear(s["x"], s["w"], s["w_scale"])}
    x = s["x"].detach().requires_grad_()
    y = fp8.linear(x, s["w"], s["w_scale"], wt=s["wt"], wt_scale=s["wt_scale"])
    grad_x, = torch.autograd.grad(y, x, s["grad"])
    return {"y": y, "grad_x": grad_x}


def _own_grouped(s):
    _, fp8 = _package()
    return {"y": fp8.grouped_matmul(s["q"], s["scale"], s["offsets"], s["w"], s["w_scale"])}


OWN = {"permute": _own_permute, "unpermute": _own_unpermute, "quantize": _own_quantize, "linear": _own_linear,
       "grouped": _own_grouped}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------ the 64-bit values
def _values(q, scale):
    """What E4M3 values with a scale per 128 columns stand for, in 64 bits."""
    column = torch.arange(q.shape[-1], device=q.device) // BLOCK
    return q.double() * scale.double()[..., column]


def _e4m3(v):
    """Nearest E4M3 value (4 significant bits, ties to even, steps of 2^-9 below 2^-6) in 64 bits."""
    exponent = torch.frexp(v)[1].clamp_min(-5)
    step = torch.ldexp(torch.ones_like(v), exponent - 4)
    return (v / step).round() * step


def _exact_quantize(v):
    q, scale = torch.empty_like(v), []
    for c in range(0, v.shape[1], BLOCK):
        part = v[:, c: c + BLOCK]
        top = part.abs().max(1, keepdim=True).values.clamp_min(AMAX_FLOOR)
        q[:, c: c + BLOCK] = _e4m3(part / (top / E4M3_MAX))
        scale.append(top / E4M3_MAX)
    return q, torch.cat(scale, 1)


def _exact_weights(w, scale):
    n = torch.arange(w.shape[-2], device=w.device) // BLOCK
    return _values(w, scale[..., n, :])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "permute":
        t, k = s["ids"].shape
        x = s["x"].double()
        route = torch.argsort(torch.where(s["ids"] < 0, case["experts"], s["ids"]).reshape(-1), stable=True)
        n = int((s["ids"] >= 0).sum())
        out = {"row_of_route": None, "offsets": None}
        if case["train"]:
            grad_x = torch.zeros_like(x)
            grad_x.index_add_(0, route[:n] // k, s["grad"][:n].double())
            out["grad_x"] = grad_x
        rows = torch.zeros(t * k, x.shape[1], dtype=torch.float64, device=x.device)
        rows[:n] = x[route[:n] // k]
        out["rows"] = rows
        if case["dtype"] == "fp8":
            scale = torch.zeros(t * k, s["scale"].shape[1], dtype=torch.float64, device=x.device)
            scale[:n] = s["scale"].double()[route[:n] // k]
            out["scale"] = scale
        return out
    if op == "unpermute":
        row, y, w = s["row_of_route"].long(), s["rows"].double(), s["weights"].double()
        total = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=y.device)
        grad_y, grad_w = torch.zeros_like(y), torch.zeros_like(w)
        for j in range(case["top_k"]):
            at = torch.nonzero(row[:, j] >= 0).flatten()
            mine = y[row[at, j]]
            total[at] += w[at, j, None] * mine
            if case["train"]:
                g = s["grad"].double()[at]
                grad_y[row[at, j]] = w[at, j, None] * g
                grad_w[at, j] = torch.einsum("th,th->t", g, mine)
        return {"out": total, "grad_rows": grad_y, "grad_weights": grad_w} if case["train"] else {"out": total}
    if op == "quantize":
        x = s["x"].double()
        if case["act"] == "none":
            q, scale = _exact_quantize(x)
            return {"q": q, "scale": scale}
        gate, up = x.split(case["width"], dim=1)
        g, u = torch.minimum(gate, torch.full_like(gate, LIMIT)), torch.clip(up, -LIMIT, LIMIT)
        sig = torch.sigmoid(g)
        q, scale = _exact_quantize(g * sig * u)
        if not case["train"]:
            return {"q": q, "scale": scale}
        d = s["grad"].double()
        dg = d * u * (sig + g * sig * (1 - sig)) * (gate <= LIMIT)
        du = d * g * sig * (up.abs() <= LIMIT)
        return {"q": q, "scale": scale, "grad_x": torch.cat([dg, du], dim=1)}
    if op == "linear":
        w = _exact_weights(s["w"], s["w_scale"])
        out = {"y": _values(*_exact_quantize(s["x"].double())) @ w.T}
        if case["train"]:
            out["grad_x"] = _values(*_exact_quantize(s["grad"].double())) @ w
        return out
    y = torch.zeros(s["q"].shape[0], case["n"], dtype=torch.float64, device="cuda")
    first = s["offsets"].tolist()
    for e in range(case["experts"]):
        a, b = first[e], first[e + 1]
        if b > a:
            y[a:b] = _values(s["q"][a:b], s["scale"][a:b]) @ _exact_weights(s["w"][e], s["w_scale"][e]).T
    return {"y": y}


# -------------------------------------------------------------------- work
def _experts_hit(case):
    """Expected number of experts with a row, the routes drawn as `_routing` draws them."""
    e, k, t = case["experts"], case["top_k"], case["tokens"] * (1 - case["drop"])
    share = [(r + 1) ** -case["skew"] for r in range(e)]
    total = sum(share)
    return sum(1 - (1 - min(1.0, k * p / total)) ** t for p in share)


def work(case):
    op = case["op"]
    if op in ("permute", "unpermute"):
        t, k, h, b = case["tokens"], case["top_k"], case["hidden"], SIZE[case["dtype"]]
        held = t * k * (1 - case["drop"])
        if op == "permute":
            move = (t + t * k) * h * b + 8 * t * k + 4 * case["experts"]
            if case["dtype"] == "fp8":
                move += (t + t * k) * 4 * -(-h // BLOCK)
            return {"bytes": move + (t + held) * h * b * case["train"], "flops": held * h * case["train"]}
        move = (t + held) * h * b + 8 * t * k
        if case["train"]:  # the rows are needed again only for the weights' gradient: counted once
            move += (t + t * k) * h * b + 4 * t * k
        return {"bytes": move, "flops": held * h * (5 if case["train"] else 2)}
    if op == "quantize":
        r, w, b = case["rows"], case["width"], SIZE[case["dtype"]]
        width_in = 2 * w if case["act"] == "swiglu" else w
        move = r * (width_in * b + w + 4 * -(-w // BLOCK))
        if case["train"]:
            move += r * (w + 2 * w) * b
        return {"bytes": move, "flops": r * w * (8 if case["act"] == "swiglu" else 2) * (2 if case["train"] else 1)}
    n, k = case["n"], case["k"]
    if op == "linear":
        t, b = case["tokens"], SIZE[case["dtype"]]
        one = t * (n + k) * b + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)
        times = 2 if case["train"] else 1
        return {"bytes": times * one, "flops": times * 2 * t * n * k}
    held = case["tokens"] * case["top_k"] * (1 - case["drop"])
    rows = case["tokens"] * case["top_k"]
    return {"bytes": held * (k + 4 * -(-k // BLOCK)) + rows * 2 * n + _experts_hit(case) * n * k,
            "flops": 2 * held * n * k}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
