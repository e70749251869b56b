"""The operators in front of and around 4-bit experts run together (``norm``, ``fp4``, ``permute``, ``experts.Fp4Experts``)
against their steps in 64 bits.

Every step but the products' f32 sums and the 16-bit roundings between them is fixed by its definition, so the steps
are followed with the operators' own quantized rows, and each result is held to its own rounding."""

from __future__ import annotations

import pytest
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.fixture(scope="module")
def ops(pkg):
    from b200moe import experts, fp4, norm, permute

    return type("Ops", (), {"experts": experts, "fp4": fp4, "norm": norm, "permute": permute})


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def routes(seed, t, k, e, drop):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ids = torch.randn(t, e, generator=g, device="cuda").topk(k, 1).indices.to(torch.int32)
    ids[torch.rand(t, k, generator=g, device="cuda") < drop] = -1
    return ids, torch.rand(t, k, generator=g, device="cuda")


def product(ops, rows, w, e, dtype):
    """64 bits of one expert's product, and the bound of its f32 sums and its rounding."""
    a = ops.fp4.dequantize(rows, torch.float32).double()
    one = ops.fp4.Weights(w.codes[e], w.scale[e], None if w.factor is None else w.factor[e: e + 1])
    b = ops.fp4.dequantize(one, torch.float32).double()
    y = a @ b.t()
    return y, a.shape[1] * 2.0**-23 * (a.abs() @ b.abs().t()) + (U[dtype] + 2.0**-22) * y.abs() + 2.0**-25


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,e,h,inter,drop", [(1, 2, 8, 256, 96, 0.0), (37, 3, 6, 320, 160, 0.2),
                                                (300, 4, 5, 512, 352, 0.0), (9, 1, 3, 128, 64, 1.0)])
def test_a_block_by_its_steps(ops, fmt, dtype, t, k, e, h, inter, drop):
    """Residual and norm, rows quantized there, experts, weighted return."""
    layer = ops.experts.Fp4Experts.from_weights(randn(1, e, 2 * inter, h) * h**-0.5, randn(2, e, h, inter) * inter**-0.5, fmt)
    x, r = randn(3, t, h, dtype=dtype), randn(4, t, h, dtype=dtype)
    gain = (1 + 0.1 * randn(5, h)).to(dtype)
    ids, weights = routes(6, t, k, e, drop)
    normed = ops.norm.rms_norm_quantize(x, gain, r, format=fmt, keep=True)
    out = layer(normed.rows, ids, weights, out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (t, h)

    p = ops.fp4.permute(normed.rows, ids, e)
    h13 = ops.fp4.grouped_matmul(p.rows, p.offsets, layer.w13, dtype)
    act = ops.fp4.swiglu_quantize(h13, 10.0, fmt)
    y = ops.fp4.grouped_matmul(act, p.offsets, layer.w2, dtype)
    off = p.offsets.tolist()
    for i in range(e):
        s = slice(off[i], off[i + 1])
        if off[i + 1] == off[i]:
            continue
        for got, rows, w in ((h13, p.rows, layer.w13), (y, act, layer.w2)):
            want, bound = product(ops, rows._replace(record=rows.record[s].contiguous()), w, i, dtype)
            assert bool(((got[s].double() - want).abs() <= bound).all())
    held = (ids >= 0)[..., None]
    parts = torch.where(held, y.double()[p.row_of_route.long().clamp_min(0)], 0.0) * weights.double()[..., None]
    want = parts.sum(1)
    bound = (k + 1) * 2.0**-23 * parts.abs().sum(1) + U[dtype] * want.abs() + 2.0**-25
    assert bool(((out.double() - want).abs() <= bound).all())
    ops.fp4.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_rows_and_their_quantized_form_give_the_same(ops, fmt):
    layer = ops.experts.Fp4Experts.from_weights(randn(1, 8, 192, 256) / 16, randn(2, 8, 256, 96) / 10, fmt)
    x = randn(3, 50, 256, dtype=torch.bfloat16)
    ids, weights = routes(4, 50, 2, 8, 0.1)
    want = layer(x, ids, weights)
    assert torch.equal(layer(ops.fp4.quantize(x, fmt), ids, weights), want)
    assert torch.equal(layer(x.float(), ids, weights), want)
    # one token at a time, the same rows by other kernels: sums in another order, then two roundings to 4 bits
    single = torch.cat([layer(x[i: i + 1], ids[i: i + 1], weights[i: i + 1]) for i in range(50)])
    off = float((single.float() - want.float()).norm() / want.float().norm())
    assert off < 2e-2  # a flipped code is off by an eighth to a half of its value, and few flip


@pytest.mark.gpu
def test_no_tokens(ops):
    layer = ops.experts.Fp4Experts.from_weights(randn(1, 4, 128, 64), randn(2, 4, 64, 64))
    ids, weights = torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda")
    assert layer(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16), ids, weights).shape == (0, 64)


@pytest.mark.gpu
def test_captured_and_replayed(ops):
    layer = ops.experts.Fp4Experts.from_weights(randn(1, 8, 256, 256) / 16, randn(2, 8, 256, 128) / 11)
    x, r, gain = randn(3, 5, 256, dtype=torch.bfloat16), randn(4, 5, 256, dtype=torch.bfloat16), torch.ones(256, device="cuda")
    ids, weights = routes(5, 5, 2, 8, 0.0)

    def step():
        return layer(ops.norm.rms_norm_quantize(x, gain, r, format="nvfp4").rows, ids, weights)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x.copy_(randn(7, 5, 256, dtype=torch.bfloat16))
    ids.copy_(routes(8, 5, 2, 8, 0.5)[0])
    g.replay()
    assert torch.equal(out, step())


@pytest.mark.gpu
def test_refusals(ops):
    cls, fp4 = ops.experts.Fp4Experts, ops.fp4
    w13, w2 = fp4.quantize_weight(randn(1, 2, 128, 64)), fp4.quantize_weight(randn(2, 2, 64, 64))
    layer = cls(w13, w2)
    x = randn(3, 4, 64, dtype=torch.bfloat16)
    ids, weights = routes(4, 4, 2, 2, 0.0)
    for bad in (lambda: cls(w2, w13), lambda: cls(w13, fp4.quantize_weight(randn(2, 2, 64, 64), "mxfp4")),
                lambda: cls(fp4.quantize_weight(randn(1, 128, 64)), w2), lambda: layer(x[:, :32].contiguous(), ids, weights),
                lambda: layer(x, ids, weights[:, :1]), lambda: layer(x.clone().requires_grad_(), ids, weights),
                lambda: layer(fp4.quantize(x, "mxfp4"), ids, weights), lambda: layer(x, ids.long(), weights)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_the_example_runs(pkg):
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("fp4_block", Path(__file__).parents[1] / "examples" / "fp4_block.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    got = mod.main(["--tokens", "64", "--hidden", "256", "--inter", "128", "--experts", "8", "--steps", "2"])
    assert got["gain_gradient"] > 0 and all(abs(v) < 1e6 for v in got.values())
