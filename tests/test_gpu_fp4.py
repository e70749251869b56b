"""The 4-bit operators (``fp4``) against their definition and plain 64-bit products.

Quantizers: every code, scale and factor is the definition's, worked out in 64 bits (16- and 32-bit values divided by
small multiples of powers of two leave no doubt there about a rounding).  Products: values are exact, so what is left
is a truncation of 2^-23 per addition times the sum of magnitudes, the two factors' products and one rounding."""

from __future__ import annotations

import pytest
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}
BLOCK = {"nvfp4": 16, "mxfp4": 32}
FORMATS = ["nvfp4", "mxfp4"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops(pkg):
    from b200moe import fp4, fp8, packing, permute

    return type("Ops", (), {"fp4": fp4, "fp8": fp8, "packing": packing, "permute": permute})


def randn(seed, *shape, dtype=torch.float32, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device).to(dtype)


# ------------------------------------------------------------- the definition
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def e2m1_codes(v):
    """Nearest code (0..7) of magnitudes, ties to the even code, 6 above."""
    grid = GRID.to(v.device)
    mid = (grid[1:] + grid[:-1]) / 2
    up = torch.searchsorted(mid, v.contiguous())  # borders below v
    tie = (up < 7) & (mid[up.clamp_max(6)] == v)
    return up + (tie & (up % 2 == 1)).long()


def e4m3_bytes(v):
    """Nearest E4M3 byte of finite values from 0 to about 448, ties to even."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v)[1].clamp_min(-5) - 4)
    r = ((v / step).round() * step).clamp(max=448.0)
    return r.float().to(torch.float8_e4m3fn).view(torch.uint8)  # exact: r is on the grid


def power_not_below(v):
    m, e = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), e - (m == 0.5).int())


def define(x, fmt, amax=None):
    """(codes 0..15 [M, K], scale bytes, factors or None) of finite rows in 64 bits."""
    x = x.double()
    b = x.view(x.shape[0], -1, BLOCK[fmt])
    top = b.abs().amax(-1)
    if fmt == "nvfp4":
        amax = x.abs().amax(1) if amax is None else amax
        factor = power_not_below(amax.clamp_min(2.0**-100) / 2688)
        scale = e4m3_bytes(top / 6 / factor[:, None])
        unit = scale.view(torch.float8_e4m3fn).double() * factor[:, None]
    else:
        factor = None
        unit = torch.where(top > 0, power_not_below(top / 6).clamp_min(2.0**-127), torch.ones_like(top))
        scale = (torch.frexp(unit)[1] + 126).to(torch.uint8)
    ratio = torch.where(unit[..., None] > 0, b.abs() / unit[..., None], torch.zeros_like(b))
    codes = e2m1_codes(ratio)
    negative = (b < 0) | ((b == 0) & torch.signbit(b) & (codes == 0))
    codes = codes + 8 * ((negative & (unit[..., None] > 0)).long())
    return codes.view(x.shape), scale, factor


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()


def values(codes, scale, factor, fmt):
    """In 64 bits, from packed bytes."""
    n = unpack(codes)
    v = GRID.to(codes.device)[n & 7] * torch.where(n > 7, -1.0, 1.0)
    s = scale.contiguous().view(torch.float8_e4m3fn).double() if fmt == "nvfp4" else \
        torch.ldexp(torch.ones(scale.shape, dtype=torch.float64, device=scale.device), scale.int() - 127)
    v = v * s.repeat_interleave(BLOCK[fmt], -1)
    return v if factor is None else v * factor.double().view(*factor.shape, *[1] * (v.dim() - factor.dim()))


def row_values(rows):
    return values(rows.codes, rows.scale, rows.factor, rows.format)


def weight_values(w):
    f = w.factor
    if f is not None and w.codes.dim() == 2:
        f = f[0]
    return values(w.codes, w.scale, f, w.format)


def same_rows(rows, x, fmt):
    codes, scale, factor = define(x, fmt)
    assert torch.equal(rows.scale, scale)
    if factor is not None:
        assert torch.equal(rows.factor.double(), factor)
    got = unpack(rows.codes)
    # the sign of a code of zero says nothing
    assert torch.equal(torch.where(got == 8, 0, got), torch.where(codes == 8, 0, codes))


# ------------------------------------------------------------------ quantizers
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,pad", [(1, 32, 0), (1, 4096, 0), (7, 96, 0), (333, 1408, 0), (64, 512, 8), (9, 544, 3),
                                     (5, 8192, 0), (3, 8224, 0), (2, 20000, 0), (4097, 64, 0)])
def test_quantize_is_the_definition(ops, fmt, dtype, m, k, pad):
    x = (randn(m + k, m, k + pad) * (1 + 20 * (randn(k, k + pad) > 2))).to(dtype)[:, pad:]
    rows = ops.fp4.quantize(x, fmt)
    same_rows(rows, x, fmt)
    for t in DTYPES:
        want = row_values(rows)
        assert torch.equal(ops.fp4.dequantize(rows, t), want.to(t) if t != torch.bfloat16 else want.bfloat16())
    again = ops.fp4.quantize(x, fmt)
    assert torch.equal(again.record, rows.record)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_ties_and_extremes(ops, fmt):
    """Every border between two codes and two scales, zeros, each type's least and largest values."""
    grid = torch.arange(0, 129, device="cuda") / 16.0  # 0 .. 8 in steps of 1/16: all borders of codes
    x = torch.zeros(64, 160, device="cuda")
    x[:, :129] = grid
    x *= torch.ldexp(torch.ones(64, device="cuda"), torch.arange(64, device="cuda") - 32)[:, None]
    x[1::2] *= -1
    for dtype in (torch.float32, torch.bfloat16):
        same_rows(ops.fp4.quantize(x.to(dtype), fmt), x.to(dtype), fmt)
    # block maxima at the borders of E4M3 scales: 6 * (odd multiple of half a step), beside a row maximum of 2688
    b = torch.zeros(1, 512, device="cuda")
    b[0, ::16] = 6 * (16 + torch.arange(32, device="cuda")) / 16.0
    b[0, 0] = 2688.0
    same_rows(ops.fp4.quantize(b, fmt), b, fmt)
    ends = torch.tensor([[3.4028234e38] * 32, [1.17549435e-38] * 32, [1e-45] * 32, [0.0] * 32, [-0.0] * 32,
                         [2.0**-100] * 32, [2.0**-101] * 32, [1e-30] * 16 + [0.0] * 16], device="cuda")
    same_rows(ops.fp4.quantize(ends, fmt), ends, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_value_that_is_no_number_spoils_its_block(ops, fmt, bad):
    x = randn(3, 5, 256)
    x[2, 77] = bad
    rows = ops.fp4.quantize(x, fmt)
    v = ops.fp4.dequantize(rows, torch.float32)
    gone = torch.zeros(5, 256, dtype=torch.bool, device="cuda")
    gone[2, slice(None) if fmt == "nvfp4" else slice(64, 96)] = True
    assert torch.equal(v.isnan(), gone)
    w = ops.fp4.quantize_weight(randn(4, 40, 256), fmt)
    for y in (ops.fp4.matmul(rows, w), ops.fp4.linear(x, w), ops.fp4.linear(x.repeat(40, 1), w)[:5],
              ops.fp4.linear(x.bfloat16(), w)):
        assert torch.equal(y.isnan().all(1), torch.tensor([0, 0, 1, 0, 0], device="cuda").bool())
        assert not y[[0, 1, 3, 4]].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,width", [(1, 32), (256, 2048), (37, 1408), (3, 96)])
def test_swiglu_quantize(ops, fmt, dtype, m, width):
    h = randn(m, m, 2 * width, dtype=dtype) * 4
    rows = ops.fp4.swiglu_quantize(h, 10.0, fmt)
    g, u = h.float()[:, :width].clamp(max=10.0), h.float()[:, width:].clamp(-10.0, 10.0)
    same_rows(rows, g / (1 + torch.exp(-g)) * u, fmt)
    g, u = h.float()[:, :width], h.float()[:, width:]
    same_rows(ops.fp4.swiglu_quantize(h, None, fmt), g / (1 + torch.exp(-g)) * u, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 32), (40, 96), (3, 17, 64), (70, 5, 1408)])
def test_quantize_weight(ops, fmt, dtype, shape):
    w = randn(sum(shape), *shape, dtype=dtype) * 0.02
    if len(shape) == 3:
        w[1] *= 100
    q = ops.fp4.quantize_weight(w, fmt)
    assert q.format == fmt
    mats = w if w.dim() == 3 else w[None]
    codes, scale = (t if w.dim() == 3 else t[None] for t in (q.codes, q.scale))
    for e, one in enumerate(mats):
        amax = one.double().abs().max().expand(one.shape[0])
        want, want_scale, factor = define(one, fmt, amax)
        assert torch.equal(scale[e], want_scale)
        if factor is not None:
            assert float(q.factor[e]) == float(factor[0])
        got = unpack(codes[e])
        assert torch.equal(torch.where(got == 8, 0, got), torch.where(want == 8, 0, want))
    assert torch.equal(ops.fp4.dequantize(q, torch.float32).double(), weight_values(q).float().double())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_of_a_pack(ops, fmt):
    """The packing kernels' codes, scales and global are weights as they are."""
    w = randn(8, 96, 512) * 0.02
    q = ops.fp4.Weights(*(ops.packing.quantize_nvfp4(w) if fmt == "nvfp4" else ops.packing.quantize_mxfp4(w)))
    x = randn(9, 21, 512, dtype=torch.bfloat16)
    check_product(ops.fp4.linear(x, q), row_values(ops.fp4.quantize(x, fmt)), weight_values(q))


# -------------------------------------------------------------------- products
def check_product(y, a, w):
    """y against a . w^T of exact values; the bound of the docstring."""
    want, mag = a @ w.t(), a.abs() @ w.abs().t()
    bound = a.shape[1] * 2.0**-23 * mag + (U[y.dtype] + 2.0**-22) * want.abs() + TINY[y.dtype]
    d = (y.double() - want).abs()
    assert bool((d <= bound).all()), f"worst excess {float((d - bound).max()):.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 32), (1, 4096, 4096), (3, 200, 96), (8, 333, 1408), (9, 129, 64), (16, 2816, 2048), (17, 2047, 608),
    (33, 4096, 320), (64, 128, 4096), (65, 4097, 1024), (128, 256, 256), (129, 257, 288), (333, 2816, 2048),
    (1000, 4096, 224), (2500, 1001, 1408), (4096, 4096, 512)])
def test_linear(ops, fmt, m, n, k):
    x = randn(m + n, m, k, dtype=torch.bfloat16)
    w = ops.fp4.quantize_weight(randn(n + k, n, k) * 0.02, fmt)
    rows = ops.fp4.quantize(x, fmt)
    a, wv = row_values(rows), weight_values(w)
    check_product(ops.fp4.linear(x, w), a, wv)
    check_product(ops.fp4.matmul(rows, w, torch.float32), a, wv)
    assert torch.equal(ops.fp4.matmul(rows, w), ops.fp4.linear(x, w))
    assert torch.equal(ops.fp4.matmul(rows, w, torch.float16), ops.fp4.linear(x, w, torch.float16))
    ops.fp4.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_linear_types_and_strides(ops, dtype, m):
    """Rows at any distance and address; a row's result does not depend on them."""
    w = ops.fp4.quantize_weight(randn(5, 264, 352) * 0.05)
    x = randn(m, m, 352, dtype=dtype)
    want = ops.fp4.linear(x, w)
    assert want.dtype == dtype
    check_product(want, row_values(ops.fp4.quantize(x)), weight_values(w))
    for pad, at in ((8, 0), (1, 0), (3, 3), (16, 8)):
        wide = torch.full((m, 352 + pad), 1e4, dtype=dtype, device="cuda")
        wide[:, at: at + 352] = x
        assert torch.equal(ops.fp4.linear(wide[:, at: at + 352], w), want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 3, 20, 300, 2500])
@pytest.mark.parametrize("k", [32, 96, 352, 512, 1408])
def test_weight_scales_at_any_address(ops, fmt, m, k):
    """Scales behind 1, 2, 4 or 8 bytes of something else, which must not be taken for theirs."""
    w = ops.fp4.quantize_weight(randn(k, 700, k) * 0.05, fmt)
    rows = ops.fp4.quantize(randn(m, m, k), fmt)
    want = ops.fp4.matmul(rows, w, torch.float32)
    check_product(want, row_values(rows), weight_values(w))
    for at in (1, 2, 4, 8):
        room = torch.full((w.scale.numel() + at + 16,), 255, dtype=torch.uint8, device="cuda")
        scale = room[at: at + w.scale.numel()].view(w.scale.shape)
        scale.copy_(w.scale)
        assert torch.equal(ops.fp4.matmul(rows, w._replace(scale=scale), torch.float32), want) or m <= 8
        check_product(ops.fp4.matmul(rows, w._replace(scale=scale), torch.float32), row_values(rows), weight_values(w))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("counts,tail,n,k", [
    ([1], 0, 128, 64), ([0, 3, 0, 17, 1, 0], 5, 200, 96), ([40, 0, 33, 64, 65], 0, 333, 352), ([1] * 300, 0, 256, 256),
    ([200, 0, 129, 1, 300], 7, 512, 640), ([5000, 1, 0, 700], 0, 2816, 288), ([0, 0, 0], 9, 130, 64),
    ([128] * 20, 0, 1024, 1408)])
def test_grouped_matmul(ops, fmt, counts, tail, n, k):
    e, s = len(counts), sum(counts) + tail
    x = randn(s, s, k)
    w = ops.fp4.quantize_weight(randn(n, e, n, k) * 0.03, fmt)
    rows = ops.fp4.quantize(x, fmt)
    off = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    a, wv = row_values(rows), weight_values(w)
    for dtype in (torch.bfloat16, torch.float32):
        y = ops.fp4.grouped_matmul(rows, off, w, dtype)
        for i in range(e):
            lo, hi = int(off[i]), int(off[i + 1])
            if hi > lo:
                check_product(y[lo:hi], a[lo:hi], wv[i])
        assert not y[s - tail:].any()
    ops.fp4.check_errors()


@pytest.mark.gpu
def test_grouped_rows_before_the_first_expert(ops):
    rows, w = ops.fp4.quantize(randn(1, 50, 64)), ops.fp4.quantize_weight(randn(2, 2, 40, 64))
    off = torch.tensor([10, 20, 45], dtype=torch.int32, device="cuda")
    y = ops.fp4.grouped_matmul(rows, off, w)
    a, wv = row_values(rows), weight_values(w)
    check_product(y[10:20], a[10:20], wv[0])
    check_product(y[20:45], a[20:45], wv[1])
    assert not y[:10].any() and not y[45:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_permute_moves_records(ops, fmt):
    x = randn(6, 37, 224, dtype=torch.bfloat16)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    ids = torch.randint(-1, 9, (37, 3), generator=g, device="cuda", dtype=torch.int32)
    rows = ops.fp4.quantize(x, fmt)
    p = ops.fp4.permute(rows, ids, 9)
    row, off = ops.permute.sort_routes(ids, 9)
    assert torch.equal(p.row_of_route, row) and torch.equal(p.offsets, off)
    held = row >= 0
    want = rows.record[:, None].expand(-1, 3, -1)
    assert torch.equal(p.rows.record[row[held].long()], want[held])
    assert not p.rows.record[~row[~held].long()].any()
    assert p.rows.columns == 224 and p.rows.format == fmt


@pytest.mark.gpu
def test_empty_rows(ops):
    w = ops.fp4.quantize_weight(randn(1, 40, 64))
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    rows = ops.fp4.quantize(x)
    assert rows.record.shape[0] == 0 and ops.fp4.dequantize(rows).shape == (0, 64)
    assert ops.fp4.linear(x, w).shape == (0, 40) and ops.fp4.matmul(rows, w).shape == (0, 40)


@pytest.mark.gpu
def test_offsets_out_of_range_are_reported(ops, pkg):
    rows, w = ops.fp4.quantize(randn(1, 20, 64)), ops.fp4.quantize_weight(randn(2, 3, 40, 64))
    ops.fp4.check_errors()
    ops.fp4.grouped_matmul(rows, torch.tensor([0, 5, 3, 30], dtype=torch.int32, device="cuda"), w)
    with pytest.raises(pkg._lib.B200MoeError):
        ops.fp4.check_errors()
    ops.fp4.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 500, 5000])
def test_graph_replay_and_another_stream(ops, m):
    w = ops.fp4.quantize_weight(randn(1, 512, 1024) * 0.02)
    x = randn(m, m, 1024, dtype=torch.bfloat16)
    want = ops.fp4.linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.fp4.linear(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    g, y = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(g):
        y = ops.fp4.linear(x, w)
    x.copy_(randn(m + 1, m, 1024, dtype=torch.bfloat16))
    g.replay()
    assert torch.equal(y, ops.fp4.linear(x, w)) and not torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_past_32_bit_offsets(ops, fmt):
    """Rows whose records, and whose own values, pass 4 GB: the last ones as by a call of their own."""
    m, k = 2_000_001, 4096
    x = torch.empty(m, k, device="cuda", dtype=torch.bfloat16)
    x[:64], x[-64:] = randn(1, 64, k), randn(2, 64, k)
    x[64:-64] = 0.0
    w = ops.fp4.quantize_weight(randn(3, 32, k) * 0.02, fmt)
    rows = ops.fp4.quantize(x, fmt)
    del x
    assert rows.record.numel() > 2**32
    y = ops.fp4.matmul(rows, w)
    for s in (slice(0, 64), slice(m - 64, m)):
        part = rows._replace(record=rows.record[s].clone())
        assert torch.equal(part.record, ops.fp4.quantize(randn(1 if s.start == 0 else 2, 64, k, dtype=torch.bfloat16), fmt).record)
        check_product(y[s], row_values(part), weight_values(w))
        assert torch.equal(ops.fp4.dequantize(rows)[s], ops.fp4.dequantize(part))
    assert not y[64:-64].any()


@pytest.mark.gpu
def test_mxfp4_scales_of_any_size(ops):
    """Rows near the ends of f32's range times ordinary weights, by each kernel; results within its normal range."""
    w = ops.fp4.quantize_weight(randn(1, 300, 256), "mxfp4")
    for m in (1, 40, 300):
        for size in (2.0**-110, 2.0**100):
            rows = ops.fp4.quantize(randn(m, m, 256) * size, "mxfp4")
            check_product(ops.fp4.matmul(rows, w, torch.float32), row_values(rows), weight_values(w))


# -------------------------------------------------------------------- refusals
@pytest.mark.gpu
def test_refusals(ops):
    f = ops.fp4
    x, w = randn(1, 8, 64, dtype=torch.bfloat16), f.quantize_weight(randn(2, 40, 64))
    w3, mx = f.quantize_weight(randn(3, 2, 40, 64)), f.quantize_weight(randn(2, 40, 64), "mxfp4")
    rows = f.quantize(x)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: f.quantize(x, "fp4"), lambda: f.quantize(x[:, :40]), lambda: f.quantize(x[:, ::2]),
                lambda: f.quantize(x.cpu()), lambda: f.quantize(x.double()), lambda: f.quantize(x[0]),
                lambda: f.quantize(torch.zeros(4, 1, device="cuda").expand(4, 64)),
                lambda: f.swiglu_quantize(x, 0.0), lambda: f.swiglu_quantize(x[:, :48]),
                lambda: f.quantize_weight(randn(1, 4, 33)), lambda: f.quantize_weight(randn(1, 0, 64)),
                lambda: f.matmul(rows, mx), lambda: f.matmul(rows, w3), lambda: f.matmul(rows._replace(columns=96), w),
                lambda: f.matmul(rows, w, torch.float64),
                lambda: f.matmul(rows, w._replace(scale=w.scale[:, :2])), lambda: f.matmul(rows, w._replace(factor=None)),
                lambda: f.matmul(rows, w._replace(factor=torch.ones(2, device="cuda"))),
                lambda: f.matmul(rows._replace(record=rows.record[:, :32]), w),
                lambda: f.matmul(f.quantize(randn(1, 8, 96)), w),
                lambda: f.grouped_matmul(rows, off, w), lambda: f.grouped_matmul(rows, off[:2], w3),
                lambda: f.grouped_matmul(rows, off.long(), w3), lambda: f.linear(x, w3), lambda: f.linear(x[:, :32], w),
                lambda: f.linear(x.clone().requires_grad_(), w), lambda: f.dequantize(rows, torch.int32),
                lambda: f.permute(rows._replace(columns=32), torch.zeros(8, 1, dtype=torch.int32, device="cuda"), 2)):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        f.linear(x.clone().requires_grad_(), w)
