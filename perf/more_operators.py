"""Cases that time and check the operators in front of 4-bit experts against plain torch forms.

The operators are the public calls of the package's ``norm`` and ``fp4`` modules:

- ``norm``      root-mean-square norm after the residual's addition (``norm.rms_norm``), with its gradients, or with
  its rows quantized in the same pass (``norm.rms_norm_quantize``: E4M3 with a scale per 128 columns, NVFP4, MXFP4);
- ``quantize``  rows, or limited SwiGLU rows, to 4-bit floating point with a scale per 16 (NVFP4) or 32 (MXFP4) columns
  (``fp4.quantize``, ``fp4.swiglu_quantize``), and the values that they stand for (``fp4.dequantize``);
- ``linear``    y = x . W^T with 4-bit operands, x quantized in the call (``fp4.linear``);
- ``grouped``   the same product of quantized rows sorted by expert with each expert's weights (``fp4.grouped_matmul``).

With ``own`` false, ``run`` computes the plain form; with ``own`` true it makes the package's calls.
"""

import math
import random

import torch

own = False

EPS = 1e-6
LIMIT = 10.0  # the framework's SwiGLU bound
E4M3_MAX, E2M1_MAX = 448.0, 6.0
AMAX_FLOOR = 1e-30  # of E4M3 blocks
FLOOR = 2.0**-100  # of NVFP4 rows
FP8_BLOCK = 128
BLOCK = {"nvfp4": 16, "mxfp4": 32}  # columns that share one scale
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one generated token in front of its experts: residual added, normed, quantized; the router reads the rows too
        {"name": "norm_token_nvfp4", "op": "norm", "rows": 1, "width": 4096, "dtype": "bf16", "residual": "same",
         "weight": "same", "out": "nvfp4", "keep": True, "train": False},
        # the largest decode batch in front of FP8 experts
        {"name": "norm_batch64_fp8", "op": "norm", "rows": 64, "width": 4096, "dtype": "bf16", "residual": "same",
         "weight": "same", "out": "fp8", "keep": False, "train": False},
        # a ragged fine-tuning batch of the smaller layer, the residual stream kept in f32
        {"name": "norm_train_ragged", "op": "norm", "rows": 1013, "width": 2048, "dtype": "f16", "residual": "f32",
         "weight": "f32", "out": "rows", "keep": False, "train": True},
        # the longest prompt of the prefill layer, forward and backward
        {"name": "norm_train_16k", "op": "norm", "rows": 16384, "width": 4096, "dtype": "bf16", "residual": "same",
         "weight": "same", "out": "rows", "keep": False, "train": True},
        # the same prompt served: rows leave the norm as NVFP4
        {"name": "norm_prefill_nvfp4", "op": "norm", "rows": 16384, "width": 4096, "dtype": "bf16",
         "residual": "same", "weight": "same", "out": "nvfp4", "keep": False, "train": False},
        # SwiGLU rows of a decode batch (32 tokens, 8 experts each) quantized for the down projection
        {"name": "swiglu_decode_nvfp4", "op": "quantize", "rows": 256, "width": 2048, "act": "swiglu",
         "format": "nvfp4", "dtype": "bf16"},
        # SwiGLU rows of a long prompt at the smaller layer's width
        {"name": "swiglu_48k_mxfp4", "op": "quantize", "rows": 49152, "width": 1408, "act": "swiglu",
         "format": "mxfp4", "dtype": "bf16"},
        # one token through a dense projection: weights streamed once
        {"name": "linear_token_nvfp4", "op": "linear", "tokens": 1, "n": 4096, "k": 4096, "format": "nvfp4",
         "dtype": "bf16"},
        # a ragged batch through the smaller layer's projection
        {"name": "linear_ragged_mxfp4", "op": "linear", "tokens": 333, "n": 2816, "k": 2048, "format": "mxfp4",
         "dtype": "bf16"},
        # a long prompt through the dense projection: tensor-bound
        {"name": "linear_8k_nvfp4", "op": "linear", "tokens": 8192, "n": 4096, "k": 4096, "format": "nvfp4",
         "dtype": "bf16"},
        # 32 decoding tokens over 384 experts: about 190 experts' weights streamed for one or two rows each
        {"name": "grouped_decode_nvfp4", "op": "grouped", "tokens": 32, "experts": 384, "top_k": 8, "n": 4096,
         "k": 4096, "format": "nvfp4", "skew": 0.0, "drop": 0.0},
        # a long prompt over the smaller layer's 64 experts, unevenly loaded: tensor-bound
        {"name": "grouped_prefill_mxfp4", "op": "grouped", "tokens": 6000, "experts": 64, "top_k": 6, "n": 2816,
         "k": 2048, "format": "mxfp4", "skew": 0.5, "drop": 0.0},
    ]


def _log(rng, lo, hi):
    """Spread over the logarithm; odd above 64, where nothing else would leave a ragged last tile."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n if n <= 64 else min(n | 1, hi)


def _thirty_twos(rng, lo, hi):
    """A width of whole blocks of 32, mostly no multiple of anything larger."""
    return 32 * (rng.randint(lo // 32, hi // 32) | 1)


def draw(rng):
    op = rng.choice(["norm", "norm", "quantize", "linear", "grouped"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    if op == "norm":
        out = rng.choice(["rows", "rows", "fp8", "nvfp4", "mxfp4"])
        train = out == "rows" and rng.random() < 0.7
        width = rng.choice([4096, 2048, _thirty_twos(rng, 64, 4000)])
        if not out.endswith("fp4") and rng.random() < 0.4:
            width = rng.randint(64, 4000) | 1
        return {"op": op, "rows": _log(rng, 1, 8192 if dtype == "f32" else 16384), "width": width, "dtype": dtype,
                "residual": rng.choice(["none", "same", "same", "f32"]), "weight": rng.choice(["same", "f32"]),
                "out": out, "keep": out != "rows" and rng.random() < 0.5, "train": train}
    if op == "quantize":
        act = rng.choice(["swiglu", "none"])
        width = rng.choice([1408, _thirty_twos(rng, 32, 1400)]) if act == "swiglu" else \
            rng.choice([1408, 2048, 4096, _thirty_twos(rng, 32, 4000)])
        return {"op": op, "rows": _log(rng, 1, 16384 if width > 1408 else 49152), "width": width, "act": act,
                "format": fmt, "dtype": dtype}
    n, k = rng.choice([(4096, 4096), (4096, 2048), (2816, 2048), (2048, 1408),
                       (rng.randint(64, 4000) | 1, _thirty_twos(rng, 128, 4000))])
    if op == "linear":
        return {"op": op, "tokens": _log(rng, 1, 8192), "n": n, "k": k, "format": fmt,
                "dtype": rng.choice(["bf16", "bf16", "f16"])}
    experts, top_k = rng.choice([(64, 6), (384, 8), (rng.randint(4, 128), rng.randint(1, 4))])
    most = 6000 * 6 * 2816 * 2048 // (n * k * top_k)  # no more work than the largest listed case
    return {"op": op, "tokens": _log(rng, 1, max(2, min(6000, most))), "experts": experts, "top_k": top_k, "n": n,
            "k": k, "format": fmt, "skew": rng.choice([0.0, 0.5]), "drop": rng.choice([0.0, 0.0, 0.1])}


# ------------------------------------------------------------------ inputs
def _activations(g, rows, width, dtype):
    """Normal values with a few wide columns, as hidden states have them."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    wide = torch.rand(width, generator=g, device="cuda") < 0.01
    return (x * torch.where(wide, 12.0, 1.0)).to(dtype)


def _routing(g, case):
    """Offsets int32 [E + 1] of the routes sorted by expert: each token takes the k largest of normal logits with a
    Zipf bias of exponent `skew`; a share `drop` of the routes has no expert and comes last."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn(t, e, generator=g, device="cuda")
    rank = torch.randperm(e, generator=g, device="cuda").float() + 1
    ids = (logits - case["skew"] * rank.log()).topk(k, dim=1).indices
    gone = torch.rand(t, k, generator=g, device="cuda") < case["drop"]
    key = torch.where(gone, e, ids).reshape(-1).sort().values
    return torch.searchsorted(key, torch.arange(e + 1, device="cuda")).to(torch.int32)


def _pack(magnitude, negative):
    """E2M1 values (magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6 and signs) as codes, two per byte, the even column low."""
    code = torch.where(magnitude < 2, magnitude * 2, torch.where(magnitude < 4, magnitude + 2, magnitude / 2 + 4))
    code = code.to(torch.uint8) | (negative.to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _record(x, fmt):
    """Quantized rows as one byte record per row, as a program holds them that got them from the quantizer: the codes,
    the scales and (NVFP4, on the next four bytes) the row's f32 factor, a power of two, padded to 16 bytes."""
    q, scale, factor = _quantize(x, fmt)
    rows, width = x.shape
    parts = [_pack(q.abs(), q < 0), _scale_bytes(scale, fmt)]
    if fmt == "nvfp4":
        parts += [torch.zeros(rows, -parts[1].shape[1] % 4, dtype=torch.uint8, device="cuda"),
                  factor[:, None].contiguous().view(torch.uint8)]
    used = sum(p.shape[1] for p in parts)
    return torch.cat(parts + [torch.zeros(rows, -used % 16, dtype=torch.uint8, device="cuda")], 1).contiguous()


def _scale_bytes(scale, fmt):
    if fmt == "nvfp4":
        return scale.to(torch.float8_e4m3fn).view(torch.uint8)
    return (torch.frexp(scale)[1] + 126).to(torch.uint8)  # 2^e as e + 127


def _weights(g, lead, n, k, fmt):
    """Weights [*lead, n, k] of N(0, 0.02): codes, scales and, NVFP4, one f32 factor per matrix."""
    count = math.prod(lead)
    codes = torch.empty((count, n, k // 2), dtype=torch.uint8, device="cuda")
    scale = torch.empty((count, n, k // BLOCK[fmt]), dtype=torch.uint8, device="cuda")
    factor = torch.empty(count, device="cuda")
    for i in range(count):
        w = 0.02 * torch.randn(n, k, generator=g, device="cuda")
        q, s, f = _quantize(w.view(1, -1), fmt)
        q = q.view(n, k)
        codes[i] = _pack(q.abs(), q < 0)
        scale[i] = _scale_bytes(s, fmt).view(n, -1)
        if fmt == "nvfp4":
            factor[i] = f[0]
    return codes.view(*lead, n, k // 2), scale.view(*lead, n, -1), factor if fmt == "nvfp4" else None


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "norm":
        rows, width, dt = case["rows"], case["width"], DTYPES[case["dtype"]]
        sum_dt = torch.float32 if case["residual"] == "f32" else dt
        s["x"] = torch.randn(rows, width, generator=g, device="cuda").to(dt)
        s["residual"] = None if case["residual"] == "none" else _activations(g, rows, width, sum_dt)
        s["weight"] = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(
            torch.float32 if case["weight"] == "f32" else dt)
        if case["train"]:
            s["grad"] = torch.randn(rows, width, generator=g, device="cuda").to(dt)
            if s["residual"] is not None:
                s["grad_sum"] = torch.randn(rows, width, generator=g, device="cuda").to(sum_dt)
    elif op == "quantize":
        width = case["width"] * (2 if case["act"] == "swiglu" else 1)
        s["x"] = _activations(g, case["rows"], width, DTYPES[case["dtype"]])
    elif op == "linear":
        s["x"] = _activations(g, case["tokens"], case["k"], DTYPES[case["dtype"]])
        s["w"] = _weights(g, (), case["n"], case["k"], case["format"])
    else:
        s["offsets"] = _routing(g, case)
        s["record"] = _record(_activations(g, case["tokens"] * case["top_k"], case["k"], torch.float32), case["format"])
        s["w"] = _weights(g, (case["experts"],), case["n"], case["k"], case["format"])
        # the plain form's padded batch: most rows of one expert
        s["most"] = max(1, int((s["offsets"][1:] - s["offsets"][:-1]).max()))
    return s


# ------------------------------------------------------------- plain forms
def _e2m1(t):
    """Nearest E2M1 magnitude, ties to the even code: steps of 0.5 below 2, 1 below 4, 2 above."""
    q = torch.where(t < 2, (t * 2).round() / 2, torch.where(t < 4, t.round(), (t / 2).round() * 2))
    return q.clamp(max=E2M1_MAX)


def _quantize(x, fmt):
    """f32 [rows, width] -> (E2M1 values with sign, block scales as f32, row factors or None)."""
    rows, width = x.shape
    b = x.reshape(rows, width // BLOCK[fmt], BLOCK[fmt])
    top = b.abs().amax(-1)
    if fmt == "mxfp4":
        mantissa, exponent = torch.frexp(top)  # the smallest e with 6 * 2^e >= top; 0 for a block of zeros
        e = torch.where(top > 0, exponent - torch.where(mantissa <= 0.75, 3, 2), 0).clamp(-127, 127)
        scale = torch.ldexp(torch.ones_like(top), e)
        q = _e2m1(torch.ldexp(b.abs(), -e[..., None]))
        return torch.where(b < 0, -q, q).view(rows, width), scale, None
    mantissa, exponent = torch.frexp(x.abs().amax(-1).clamp_min(FLOOR))  # the smallest 2^e with 6 * 448 * 2^e >= amax
    factor = torch.ldexp(torch.ones_like(mantissa), exponent - torch.where(mantissa <= 2688 / 4096, 12, 11))
    six = torch.full_like(factor, E2M1_MAX)  # a quotient with a plain number would be a product with its reciprocal
    scale = (top / (six * factor)[:, None]).to(torch.float8_e4m3fn).float()
    unit = scale * factor[:, None]
    t = torch.where((unit > 0)[..., None], b.abs() / unit[..., None], torch.zeros_like(b))
    q = _e2m1(t)
    return torch.where(b < 0, -q, q).view(rows, width), scale, factor


def _values(q, scale, factor, fmt):
    """What quantized rows stand for, in f32."""
    v = (q.view(*scale.shape, BLOCK[fmt]) * scale[..., None]).view(q.shape)
    return v if factor is None else v * factor[..., None]


def _unpack(codes, scale, fmt):
    """Codes [..., K / 2] and scale bytes -> f32 values without the factor."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    pairs = torch.stack([grid.repeat(16), grid.repeat_interleave(16)], 1)  # both values of a byte
    s = scale.contiguous().view(torch.float8_e4m3fn).float() if fmt == "nvfp4" else \
        torch.ldexp(torch.ones(scale.shape, device=scale.device), scale.int() - 127)
    q = pairs[codes.int()].view(*codes.shape[:-1], -1, BLOCK[fmt])
    return q.mul_(s[..., None]).view(*codes.shape[:-1], -1)


def _weight_values(w, fmt):
    codes, scale, factor = w
    v = _unpack(codes, scale, fmt)
    return v if factor is None else v.mul_(factor.view(-1, *[1] * (v.dim() - 1)) if v.dim() == 3 else factor)


def _record_parts(record, k, fmt):
    """(codes, scales, factors) of a record of quantized rows."""
    codes, at = record[:, : k // 2], k // 2 + k // BLOCK[fmt]
    scale = record[:, k // 2: at]
    if fmt == "mxfp4":
        return codes, scale, None
    at += -at % 4
    return codes, scale, record[:, at: at + 4].contiguous().view(torch.float32)[:, 0]


def _plain_norm(s):
    case, w = s["case"], s["weight"].float()
    dt = DTYPES[case["dtype"]]
    out = {}
    if s["residual"] is None:
        h = s["x"].float()
    else:  # the norm is that of the sum as stored
        out["sum"] = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
        h = out["sum"].float()
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    y = h * rstd * w
    if case["out"] == "rows" or case["keep"]:
        out["y"] = y.to(dt)
    if case["out"] == "fp8":
        rows, width = y.shape
        b = torch.cat([y, y.new_zeros(rows, -width % FP8_BLOCK)], 1).view(rows, -1, FP8_BLOCK)
        amax = b.abs().amax(-1).clamp_min(AMAX_FLOOR)
        top = torch.full_like(amax, E4M3_MAX)
        out["q"] = (b * (top / amax)[..., None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :width].contiguous()
        out["scale"] = amax / top
    elif case["out"] != "rows":
        out["values"] = _values(*_quantize(y, case["out"]), case["out"]).to(torch.bfloat16)
    if case["train"]:
        d = s["grad"].float()
        unit = h * rstd
        g = d * w
        grad = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
        if s["residual"] is not None:
            grad = grad + s["grad_sum"].float()
            out["grad_residual"] = grad.to(s["residual"].dtype)
        out["grad_x"] = grad.to(dt)
        out["grad_weight"] = (d * unit).sum(0).to(s["weight"].dtype)
    return out


def _plain_quantize(s):
    case, x = s["case"], s["x"].float()
    if case["act"] == "swiglu":
        g, u = x[:, : case["width"]].clamp(max=LIMIT), x[:, case["width"]:].clamp(-LIMIT, LIMIT)
        x = g / (1 + torch.exp(-g)) * u
    return {"values": _values(*_quantize(x, case["format"]), case["format"]).to(torch.bfloat16)}


def _plain_linear(s):
    fmt, x = s["case"]["format"], s["x"]
    return {"y": (_values(*_quantize(x.float(), fmt), fmt) @ _weight_values(s["w"], fmt).t()).to(x.dtype)}


def _plain_grouped(s):
    case, off, fmt = s["case"], s["offsets"].long(), s["case"]["format"]
    codes, scale, factor = _record_parts(s["record"], case["k"], fmt)
    v = _unpack(codes, scale, fmt)
    v = v if factor is None else v * factor[:, None]
    at = torch.arange(v.shape[0], device=v.device)
    expert = torch.searchsorted(off[1:].contiguous(), at, right=True).clamp_max(case["experts"] - 1)
    held = (at < off[-1])[:, None]
    place = (at - off[expert]).clamp_max(s["most"])  # rows without an expert go to a place of their own
    x = v.new_zeros((case["experts"], s["most"] + 1, case["k"]))
    x[expert, place] = torch.where(held, v, 0.0)
    y = x[:, : s["most"]] @ _weight_values(s["w"], fmt).transpose(1, 2)
    y = torch.where(held, y[expert, place.clamp_max(s["most"] - 1)], 0.0)
    return {"y": y.to(torch.bfloat16)}


PLAIN = {"norm": _plain_norm, "quantize": _plain_quantize, "linear": _plain_linear, "grouped": _plain_grouped}


# ---------------------------------------------------------- the package's calls
def _package():
    from __graft_entry__ import load_package

    load_package()
    from b200moe import fp4, norm

    return norm, fp4


def _own_norm(s):
    norm, fp4 = _package()
    case = s["case"]
    if case["out"] == "rows":
        if not case["train"]:
            y, total = norm.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
            return {"y": y} if total is None else {"sum": total, "y": y}
        x, w = s["x"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
        if s["residual"] is None:
            y, _ = norm.rms_norm(x, w, eps=EPS)
            grad_x, grad_w = torch.autograd.grad(y, (x, w), s["grad"])
            return {"y": y, "grad_x": grad_x, "grad_weight": grad_w}
        r = s["residual"].detach().requires_grad_()
        y, total = norm.rms_norm(x, w, r, eps=EPS)
        grad_x, grad_r, grad_w = torch.autograd.grad((y, total), (x, r, w), (s["grad"], s["grad_sum"]))
        return {"sum": total, "y": y, "grad_x": grad_x, "grad_residual": grad_r, "grad_weight": grad_w}
    rows, total, y = norm.rms_norm_quantize(s["x"], s["weight"], s["residual"], eps=EPS, format=case["out"],
                                            keep=case["keep"])
    out = {"q": rows[0], "scale": rows[1]} if case["out"] == "fp8" else {"values": fp4.dequantize(rows)}
    if total is not None:
        out["sum"] = total
    if y is not None:
        out["y"] = y
    return out


def _own_quantize(s):
    _, fp4 = _package()
    case = s["case"]
    if case["act"] == "swiglu":
        return {"values": fp4.dequantize(fp4.swiglu_quantize(s["x"], limit=LIMIT, format=case["format"]))}
    return {"values": fp4.dequantize(fp4.quantize(s["x"], format=case["format"]))}


def _own_linear(s):
    _, fp4 = _package()
    return {"y": fp4.linear(s["x"], fp4.Weights(*s["w"]))}


def _own_grouped(s):
    _, fp4 = _package()
    case = s["case"]
    rows = fp4.Rows(s["record"], case["k"], case["format"])
    return {"y": fp4.grouped_matmul(rows, s["offsets"], fp4.Weights(*s["w"]))}


OWN = {"norm": _own_norm, "quantize": _own_quantize, "linear": _own_linear, "grouped": _own_grouped}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------ the 64-bit values
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_e2m1(v):
    """Nearest E2M1 value by counting the borders below it; a border goes to the even code."""
    mag, out = v.abs(), torch.zeros_like(v)
    for i in range(7):
        border = (GRID[i] + GRID[i + 1]) / 2
        over = mag >= border if i % 2 else mag > border
        out += over * (GRID[i + 1] - GRID[i])
    return torch.copysign(out, v)


def _exact_e4m3(v):
    """Nearest E4M3 value (4 significant bits, ties to even, steps of 2^-9 below 2^-6)."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v)[1].clamp_min(-5) - 4)
    return ((v / step).round() * step).clamp(max=E4M3_MAX)


def _power(v):
    """The smallest power of two that is not below v."""
    m, e = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), e - (m == 0.5).int())


def _exact_quantized(v, fmt):
    """The values that quantized rows stand for, a block of columns at a time."""
    out = torch.empty_like(v)
    whole = _power(v.abs().max(1, keepdim=True).values.clamp_min(FLOOR) / (E2M1_MAX * E4M3_MAX))
    size = BLOCK[fmt]
    parts = v.unfold(1, size, size)
    top = parts.abs().max(2, keepdim=True).values
    if fmt == "nvfp4":
        unit = _exact_e4m3(top / E2M1_MAX / whole[..., None]) * whole[..., None]
    else:
        unit = _power(top / E2M1_MAX) * (top > 0)
    ratio = torch.where(unit > 0, parts / unit, torch.zeros_like(parts))
    out.copy_((_exact_e2m1(ratio) * unit).reshape(v.shape))
    return out


def _exact_codes(codes, scale, factor, fmt):
    low, high = (codes & 15).int(), (codes >> 4).int()
    nibble = torch.stack([low, high], -1).flatten(-2)
    e, m = (nibble >> 1) & 3, (nibble & 1).double()
    v = torch.where(e > 0, torch.ldexp(1 + m / 2, e - 1), m / 2) * torch.where(nibble > 7, -1.0, 1.0)
    b = scale.int()
    if fmt == "nvfp4":
        se, sm = (b >> 3) & 15, (b & 7).double() / 8
        sc = torch.where(se > 0, torch.ldexp(1 + sm, se - 7), torch.ldexp(sm, torch.full_like(se, -6)))
    else:
        sc = torch.ldexp(torch.ones(b.shape, dtype=torch.float64, device=b.device), b - 127)
    v = v * sc.repeat_interleave(BLOCK[fmt], -1)
    return v if factor is None else v * factor.double().reshape(-1, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        out = {}
        x, w = s["x"].double(), s["weight"].double().requires_grad_(case["train"])
        if s["residual"] is not None:
            out["sum"] = x + s["residual"].double()
            x = out["sum"].to(s["residual"].dtype).double()  # stored, then normed
        x.requires_grad_(case["train"])
        y = x * torch.rsqrt(x.square().sum(1, keepdim=True) / x.shape[1] + EPS) * w
        if case["out"] == "rows" or case["keep"]:
            out["y"] = y.detach()
        if case["out"] == "fp8":
            q, scale = torch.empty_like(y), []
            for c in range(0, y.shape[1], FP8_BLOCK):
                part = y[:, c: c + FP8_BLOCK]
                top = part.abs().max(1, keepdim=True).values.clamp_min(AMAX_FLOOR) / E4M3_MAX
                q[:, c: c + FP8_BLOCK] = torch.copysign(_exact_e4m3(part.abs() / top), part)
                scale.append(top)
            out["q"], out["scale"] = q, torch.cat(scale, 1)
        elif case["out"] != "rows":
            out["values"] = _exact_quantized(y, case["out"])
        if case["train"]:
            grad_x, out["grad_weight"] = torch.autograd.grad(y, (x, w), s["grad"].double())
            if s["residual"] is not None:
                grad_x = grad_x + s["grad_sum"].double()
                out["grad_residual"] = grad_x
            out["grad_x"] = grad_x
        return out
    if op == "quantize":
        v = s["x"].double()
        if case["act"] == "swiglu":
            gate, up = v.split(case["width"], 1)
            gate = torch.minimum(gate, torch.full_like(gate, LIMIT))
            v = gate * torch.sigmoid(gate) * torch.clip(up, -LIMIT, LIMIT)
        return {"values": _exact_quantized(v, case["format"])}
    codes, scale, factor = s["w"]
    if op == "linear":
        x = _exact_quantized(s["x"].double(), case["format"])
        return {"y": x @ _exact_codes(codes, scale, factor, case["format"]).T}
    x = _exact_codes(*_record_parts(s["record"], case["k"], case["format"]), case["format"])
    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device="cuda")
    first = s["offsets"].tolist()
    for e in range(case["experts"]):
        a, b = first[e], first[e + 1]
        if b > a:
            one = None if factor is None else factor[e: e + 1]
            y[a:b] = x[a:b] @ _exact_codes(codes[e], scale[e], one, case["format"]).T
    return {"y": y}


# -------------------------------------------------------------------- work
def _experts_hit(case):
    """Expected number of experts with a row, the routes drawn as `_routing` draws them."""
    e, k, t = case["experts"], case["top_k"], case["tokens"] * (1 - case["drop"])
    share = [(r + 1) ** -case["skew"] for r in range(e)]
    total = sum(share)
    return sum(1 - (1 - min(1.0, k * p / total)) ** t for p in share)


def _packed(width, fmt):
    """Bytes of a quantized row."""
    return width / 2 + width / BLOCK[fmt] + (4 if fmt == "nvfp4" else 0)


def work(case):
    op = case["op"]
    if op == "norm":
        r, w, b = case["rows"], case["width"], SIZE[case["dtype"]]
        rb = 0 if case["residual"] == "none" else 4 if case["residual"] == "f32" else b
        move = b + 2 * rb + (b if case["out"] == "rows" or case["keep"] else 0)
        total = r * w * move + w * b
        if case["out"] == "fp8":
            total += r * (w + 4 * -(-w // FP8_BLOCK))
        elif case["out"] != "rows":  # written, and read back as 16-bit values
            total += r * (2 * _packed(w, case["out"]) + 2 * w)
        if case["train"]:  # the stored sum and both gradients in, the inputs' gradients out
            total += r * w * (2 * b + (rb if rb else b) + rb + (rb if rb and rb != b else 0)) + 2 * w * b
        return {"bytes": total, "flops": r * w * (6 + 8 * case["train"])}
    if op == "quantize":
        r, w, b = case["rows"], case["width"], SIZE[case["dtype"]]
        width_in = 2 * w if case["act"] == "swiglu" else w
        return {"bytes": r * (width_in * b + 2 * _packed(w, case["format"]) + 2 * w),
                "flops": r * w * (9 if case["act"] == "swiglu" else 3)}
    n, k = case["n"], case["k"]
    matrix = n * (k / 2 + k / BLOCK[case["format"]])
    if op == "linear":
        t, b = case["tokens"], SIZE[case["dtype"]]
        return {"bytes": t * (n + k) * b + matrix, "flops": 2 * t * n * k}
    rows = case["tokens"] * case["top_k"]
    held = rows * (1 - case["drop"])
    return {"bytes": held * _packed(k, case["format"]) + rows * 2 * n + _experts_hit(case) * matrix,
            "flops": 2 * held * n * k}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
