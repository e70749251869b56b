"""The 4-bit operators (``fp4``, ``experts.Fp4Experts``) where they are easiest to get wrong: scales and factors at the ends
of f32, every kernel's own range of rows and columns, gradients that have no way back, offsets that fall, two streams.

Products: a truncation of 2^-23 per addition times the sum of magnitudes, the factors' products and one rounding, as
in ``test_gpu_fp4``; where values are small integers every partial sum is one below 2^24 and the product is exact."""

from __future__ import annotations

import pytest
import torch
from test_gpu_fp4 import FORMATS, check_product, ops, randn, row_values, weight_values  # noqa: F401
from test_gpu_fp4_experts import test_a_block_by_its_steps as block_by_steps


# ----------------------------------------------------------- the ends of f32
@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 40, 300, 2500])
@pytest.mark.parametrize("rows_size,factor", [(2.0**122, None), (2.0**122, 3.1e-9), (2.0**-95, 1.3e-11), (2.0**-60, 7e30),
                                              (2.0**90, 1.7e-33)])
def test_nvfp4_factors_of_any_size(ops, m, rows_size, factor):  # noqa: F811
    """Rows near the ends of f32 times a matrix factor (None: 0.02's, a power of two) that brings results back: no kernel may
    pass f32 on the way (sums reach 2^24 before their factors)."""
    w = ops.fp4.quantize_weight(randn(1, 300, 256) * 0.02)
    if factor is not None:
        w = w._replace(factor=torch.full_like(w.factor, factor))
    x = randn(m, m, 256) * rows_size
    rows = ops.fp4.quantize(x)
    a, wv = row_values(rows), weight_values(w)
    assert 2.0**-126 < float((a @ wv.t()).abs().max()) < 3e38
    check_product(ops.fp4.matmul(rows, w, torch.float32), a, wv)
    check_product(ops.fp4.linear(x, w), a, wv)
    y = ops.fp4.grouped_matmul(rows, torch.tensor([0, m], dtype=torch.int32, device="cuda"),
                               w._replace(codes=w.codes[None], scale=w.scale[None]), torch.float32)
    check_product(y, a, wv)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 4, 40, 300])
@pytest.mark.parametrize("weights_size,rows_size", [(2.0**122, 2.0**-60), (2.0**122, 2.0**-110), (2.0**-110, 2.0**100),
                                                    (2.0**124, 2.0**-20), (2.0**-115, 2.0**122)])
def test_mxfp4_scales_of_both_sides(ops, m, weights_size, rows_size):  # noqa: F811
    """Scales of weights and rows near opposite ends of f32: the product of a block's sum with one of them alone passes it."""
    w = ops.fp4.quantize_weight(randn(1, 300, 256) * weights_size, "mxfp4")
    rows = ops.fp4.quantize(randn(m, m, 256) * rows_size, "mxfp4")
    check_product(ops.fp4.matmul(rows, w, torch.float32), row_values(rows), weight_values(w))


@pytest.mark.gpu
def test_mxfp4_scales_that_are_no_number(ops):  # noqa: F811
    """A NaN scale on either side, by few rows' kernel and by the tiles': its rows and columns, and nothing else."""
    for m in (2, 40):
        w = ops.fp4.quantize_weight(randn(1, 50, 256), "mxfp4")
        w.scale[7, 3] = 255
        rows = ops.fp4.quantize(randn(m, m, 256), "mxfp4")
        rows.scale[1, 5] = 255
        gone = ops.fp4.matmul(rows, w).isnan()
        want = torch.zeros(m, 50, dtype=torch.bool, device="cuda")
        want[1], want[:, 7] = True, True
        assert torch.equal(gone, want)


# ------------------------------------------------------------- gradients lost
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_what_has_no_gradient_refuses_it(ops, fmt):  # noqa: F811
    """Tokens or router weights that require a gradient, whatever form the tokens come in; under no_grad all serve."""
    from b200moe.experts import Fp4Experts

    layer = Fp4Experts.from_weights(randn(1, 4, 128, 64, dtype=torch.bfloat16).requires_grad_(), randn(2, 4, 64, 64), fmt)
    x = randn(3, 6, 64, dtype=torch.bfloat16)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    ids = torch.randint(0, 4, (6, 2), generator=g, device="cuda", dtype=torch.int32)
    weights, rows = torch.rand(6, 2, generator=g, device="cuda"), ops.fp4.quantize(x, fmt)
    want = layer(x, ids, weights)
    learned, leaf = weights.clone().requires_grad_(), x.clone().requires_grad_()
    for bad in (lambda: layer(rows, ids, learned), lambda: layer(x, ids, learned), lambda: layer(leaf, ids, weights),
                lambda: ops.fp4.quantize(leaf, fmt), lambda: ops.fp4.swiglu_quantize(leaf, 10.0, fmt)):
        with pytest.raises(ValueError, match="gradient"):
            bad()
    with torch.no_grad():
        assert torch.equal(layer(rows, ids, learned), want) and torch.equal(layer(leaf, ids, learned), want)
        assert torch.equal(ops.fp4.quantize(leaf, fmt).record, rows.record)
        ops.fp4.swiglu_quantize(leaf, 10.0, fmt)


# ------------------------------------------------------------------ values back
def once(v, dtype):
    """64-bit values rounded once to bf16 or f16 (torch's own conversion passes through f32)."""
    bits, least = (8, -133) if dtype == torch.bfloat16 else (11, -24)
    e = (torch.frexp(v)[1] - bits).clamp_min(least)
    return torch.ldexp(torch.ldexp(v, -e).round(), e).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("low,high", [(1e-4, 1.0), (1e-10, 1e-6), (1e-40, 1e-36)])
def test_values_of_any_factor_are_rounded_once(ops, dtype, low, high):  # noqa: F811
    """Factors of 24 bits, as a pack's: products of 30 bits, of which some round in f32 to a border of 16-bit values: one in
    2^14 for f16, in 2^17 for bf16."""
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    e, n, k = 4096, 8, 256
    factor = torch.exp(torch.rand(e, generator=g, device="cuda", dtype=torch.float64) *
                       torch.log(torch.tensor(high / low, dtype=torch.float64)).item() +
                       torch.log(torch.tensor(low, dtype=torch.float64)).item()).float()
    codes = torch.randint(0, 256, (e, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.randint(0, 127, (e, n, k // 16), generator=g, device="cuda", dtype=torch.uint8)
    w = ops.fp4.Weights(codes, scale, factor)
    want = once(weight_values(w), dtype)
    assert torch.equal(ops.fp4.dequantize(w, dtype), want)


# ------------------------------------------------------------- offsets that fall
@pytest.mark.gpu
@pytest.mark.parametrize("which", FORMATS + ["fp8"])
@pytest.mark.parametrize("c", [1, 2, 5, 20])  # rows per expert by which another kernel is chosen
@pytest.mark.parametrize("offsets,held", [([0, 30, 10, 50], [(0, 0, 30)]), ([0, 30, 40, 10], [(0, 0, 30), (1, 30, 40)]),
                                          ([10, 5, 20, 30], [(2, 20, 30)]), ([0, 60, 0, 60], [(0, 0, 60)]),
                                          ([5, 20, 70, 40], [(0, 5, 20)]), ([-10, 20, 15, 40], [(2, 15, 40)]),
                                          ([0, 20, 10, 30], [(0, 0, 20)])])
def test_offsets_that_fall(ops, pkg, which, c, offsets, held):  # noqa: F811
    """Experts whose rows lie in order keep their results: a later expert that goes back over them, or the rows behind the last
    offset, must not write there.  Rows before the first offset are zeros."""
    n, k, s = 200, 96, 60 * c
    x, w = randn(c, s, k), randn(2, 3, n, k)
    if which == "fp8":
        q, wq = ops.fp8.quantize(x), ops.fp8.quantize_weight(w)
        run = lambda off: ops.fp8.grouped_matmul(*q, off, *wq)  # noqa: E731
        one = lambda e, a, b: ops.fp8.grouped_matmul(*q, good(e, a, b), *wq)  # noqa: E731
    else:
        q, wq = ops.fp4.quantize(x, which), ops.fp4.quantize_weight(w, which)
        run = lambda off: ops.fp4.grouped_matmul(q, off, wq)  # noqa: E731
        one = lambda e, a, b: ops.fp4.grouped_matmul(q, good(e, a, b), wq)  # noqa: E731

    def good(e, a, b):
        return torch.tensor([a] * (e + 1) + [b] * (3 - e), dtype=torch.int32, device="cuda")

    want = [(c * a, c * b, one(e, c * a, c * b)[c * a: c * b]) for e, a, b in held]
    ops.fp4.check_errors()
    y = run(torch.tensor([c * o for o in offsets], dtype=torch.int32, device="cuda"))
    for a, b, rows in want:
        assert torch.equal(y[a:b], rows) and rows.any()
    assert not y[: max(0, c * offsets[0])].any()
    with pytest.raises(pkg._lib.B200MoeError):
        ops.fp4.check_errors()
    ops.fp4.check_errors()


# ------------------------------------------------- each kernel's rows and columns
def integers(seed, *shape):
    """E2M1's integers, a 6 in each block of 16: quantizing leaves them as they are."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.tensor([0.0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device="cuda")[
        torch.randint(0, 11, shape, generator=g, device="cuda")]
    x[..., ::16] = 6.0
    return x


def check_exact(ops, fmt, m, n, k):  # noqa: F811
    """Sums stay below 36 * 2^14 < 2^24: whatever their order, a product is the integer."""
    assert 36 * k < 2**24
    x, w = integers(m + k, m, k), integers(n + k, n, k)
    rows, q = ops.fp4.quantize(x, fmt), ops.fp4.quantize_weight(w, fmt)
    assert torch.equal(ops.fp4.dequantize(rows, torch.float32), x) and torch.equal(ops.fp4.dequantize(q, torch.float32), w)
    want = (x.double() @ w.double().t()).float()
    assert torch.equal(ops.fp4.matmul(rows, q, torch.float32), want)
    assert torch.equal(ops.fp4.linear(x.bfloat16(), q, torch.float32), want)
    assert torch.equal(ops.fp4.linear(x, q), want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 2, 3, 8])
@pytest.mark.parametrize("n,k", [(333, 32), (65, 1056), (333, 2048), (333, 2080), (64, 4064), (333, 4096), (333, 4128), (120, 7168),
                                 (17, 8224), (333, 14336), (2368, 6144)])
def test_few_rows_are_exact(ops, fmt, m, n, k):  # noqa: F811
    """Four warps and eight along K, blocks that end inside, more blocks than a warp has in flight (K above 4096), rows that
    fill shared memory (8 x 7168, 3 x 14336), one row tile more than the GPU has SMs."""
    check_exact(ops, fmt, m, n, k)
    ops.fp4.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,k", [(2, 2048), (4, 1024), (8, 512), (3, 1312), (5, 800), (7, 96), (8, 32), (1, 4064)])
def test_few_rows_quantized_by_the_product(ops, fmt, m, k):  # noqa: F811
    """Up to 4096 values, by the pieces of 16 that whole warps, or not, share with a row; two rows of very different size."""
    check_exact(ops, fmt, m, 100, k)
    x, w = randn(m, m, k, dtype=torch.bfloat16), ops.fp4.quantize_weight(randn(k, 100, k), fmt)
    x[-1] *= 1000
    check_product(ops.fp4.linear(x, w), row_values(ops.fp4.quantize(x, fmt)), weight_values(w))
    assert torch.equal(ops.fp4.linear(x, w), ops.fp4.matmul(ops.fp4.quantize(x, fmt), w))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(16, 520, 4128), (40, 2000, 4128), (100, 520, 14336), (200, 4096, 7168), (1000, 520, 6144),
                                   (3000, 1000, 4128), (9, 8192, 2080)])
def test_more_rows_are_exact(ops, fmt, m, n, k):  # noqa: F811
    check_exact(ops, fmt, m, n, k)
    ops.fp4.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("counts,tail,n,k", [
    ([60, 0, 128, 129, 1], 0, 333, 352), ([100, 90, 130, 127, 65], 20, 512, 1408), ([53], 0, 100, 64), ([0, 0, 0, 440], 3, 1000, 4128),
    ([70] * 40, 0, 256, 608)])
def test_grouped_rows_of_128_are_exact(ops, fmt, dtype, counts, tail, n, k):  # noqa: F811
    """52 to 112 rows per matrix: the kernel with 128 of them as the MMA's M."""
    e, s = len(counts), sum(counts) + tail
    assert 52 * e < s <= 112 * e
    x, w = integers(s, s, k), integers(n, e, n, k)
    off = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    y = ops.fp4.grouped_matmul(ops.fp4.quantize(x, fmt), off, ops.fp4.quantize_weight(w, fmt), dtype)
    for i in range(e):
        lo, hi = int(off[i]), int(off[i + 1])
        assert torch.equal(y[lo:hi], (x[lo:hi].double() @ w[i].double().t()).float().to(dtype))
    assert not y[s - tail:].any()
    ops.fp4.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,k,e", [(50, 3, 5), (100, 4, 5), (400, 4, 5), (6, 5, 3)])
def test_a_block_by_every_kernel(pkg, fmt, t, k, e):
    """30, 80, 320 and 10 rows per expert (in the last, tokens name experts twice)."""
    from b200moe import experts, fp4, norm, permute

    every = type("Ops", (), {"experts": experts, "fp4": fp4, "norm": norm, "permute": permute})
    if k <= e:
        return block_by_steps(every, fmt, torch.bfloat16, t, k, e, 512, 352, 0.0)
    layer = experts.Fp4Experts.from_weights(randn(1, e, 128, 64) / 8, randn(2, e, 64, 64) / 8, fmt)
    x, weights = randn(3, t, 64, dtype=torch.bfloat16), torch.rand(t, k, device="cuda")
    ids = (torch.arange(t * k, device="cuda").view(t, k) % e).to(torch.int32)
    parts = torch.stack([layer(x, ids[:, i: i + 1].contiguous(), torch.ones(t, 1, device="cuda"), torch.float32)
                         for i in range(k)], 1).double() * weights.double()[..., None]
    bound = 2.0**-8 * parts.sum(1).abs() + (k + 1) * 2.0**-23 * parts.abs().sum(1)
    assert bool(((layer(x, ids, weights).double() - parts.sum(1)).abs() <= bound).all())


# ------------------------------------------------------------------ two streams
@pytest.mark.gpu
@pytest.mark.parametrize("what", ["linear_1", "linear_40", "linear_5000", "grouped"])
def test_calls_on_two_streams_at_once(ops, what):  # noqa: F811
    """Alternating calls with inputs of their own, nothing waiting in between: each result is the one of a call alone."""
    w = ops.fp4.quantize_weight(randn(1, 4, 1024, 2048) * 0.02)
    one = w._replace(codes=w.codes[0], scale=w.scale[0], factor=w.factor[:1])
    if what == "grouped":
        xs = [ops.fp4.quantize(randn(i, 300, 2048)) for i in range(6)]
        offs = [torch.tensor([0, 10 * i, 100, 250 + i, 300], dtype=torch.int32, device="cuda") for i in range(6)]
        run = lambda i: ops.fp4.grouped_matmul(xs[i], offs[i], w)  # noqa: E731
    else:
        xs = [randn(i, int(what[7:]), 2048, dtype=torch.bfloat16) for i in range(6)]
        run = lambda i: ops.fp4.linear(xs[i], one)  # noqa: E731
    want = [run(i) for i in range(6)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for j in range(60):
        with torch.cuda.stream(streams[j % 2]):
            got.append((j % 6, run(j % 6)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])
    ops.fp4.check_errors()
