"""The FP8 expert path's operators (``permute``, ``fp8``, ``experts``) against plain 64-bit forms.

Tolerances follow from the arithmetic: ``half_ulp`` of the stored type for the one
rounding, and for f32 sums a term of 2^-23 per addition times the sum of magnitudes
(an addition that truncates loses at most that much of its running sum)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(pkg):
    from b200moe import experts, fp8, permute

    return type("Ops", (), {"permute": permute, "fp8": fp8, "experts": experts})


def rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def routes(g, t, k, e, drop=0.0, skew=0.0):
    logits = randn(g, t, e) - skew * torch.log1p(torch.arange(e, device="cuda").float())
    ids = logits.topk(min(k, e), 1).indices.to(torch.int32)
    if k > e:  # more slots than experts: repeated ids
        ids = torch.randint(0, e, (t, k), generator=g, device="cuda", dtype=torch.int32)
    if drop:
        ids[torch.rand(t, k, generator=g, device="cuda") < drop] = -1
    return ids


def sorted_rows(ids, e):
    """numpy: row_of_route and offsets of the stable sort."""
    flat = ids.cpu().numpy().reshape(-1)
    key = np.where((flat < 0) | (flat >= e), e, flat)
    order = np.argsort(key, kind="stable")
    row = np.empty(len(flat), np.int64)
    row[order] = np.arange(len(flat))
    row = np.where(key == e, ~row, row)
    return row.reshape(ids.shape).astype(np.int32), np.searchsorted(key[order], np.arange(e + 1)).astype(np.int32)


def within(got, want, bound):
    """|got - want| <= bound everywhere, where want is finite."""
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), f"worst excess {float((d - bound).max()):.3e}"


# -------------------------------------------------------------------- permute
@pytest.mark.gpu
@pytest.mark.parametrize("t,k,e,drop", [
    (1, 8, 384, 0.0), (1, 1, 1, 0.0), (3, 2, 1024, 0.0), (7, 6, 64, 0.5), (257, 8, 384, 0.0), (256, 8, 5, 0.1),
    (341, 6, 64, 0.0), (342, 6, 64, 1.0), (1013, 6, 64, 0.1), (4096, 8, 384, 0.05), (2049, 1, 1024, 0.0),
    (5, 70, 9, 0.2), (9001, 3, 33, 0.3)])
def test_sort_routes(ops, t, k, e, drop):
    ids = routes(rng(t), t, k, e, drop)
    if drop == 0.5:  # every id that is not an expert's, at both ends
        ids[0, 0], ids[1, 0], ids[2, 0] = e, 2**31 - 1, -(2**31)
    row, offsets = ops.permute.sort_routes(ids, e)
    want_row, want_offsets = sorted_rows(ids, e)
    assert np.array_equal(offsets.cpu().numpy(), want_offsets)
    assert np.array_equal(row.cpu().numpy(), want_row)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, E4M3])
@pytest.mark.parametrize("t,k,e,h,drop,stride", [
    (1, 8, 384, 4096, 0.0, 0), (37, 6, 64, 2048, 0.3, 0), (64, 8, 384, 1001, 0.0, 0), (300, 4, 16, 100, 0.1, 0),
    (33, 2, 8, 256, 0.2, 8), (33, 2, 8, 256, 0.2, 3), (5, 3, 4, 1, 0.0, 0)])
def test_permute_moves_rows(ops, dtype, t, k, e, h, drop, stride):
    g = rng(h + t)
    x = randn(g, t, h + stride).clamp(-400, 400).to(dtype)[:, :h]
    ids = routes(g, t, k, e, drop)
    scale = torch.rand(t, 5, generator=g, device="cuda") if dtype == E4M3 else None
    p = ops.permute.permute(x, ids, e, scale=scale)
    row, offsets = sorted_rows(ids, e)
    want = np.zeros((t * k, h), np.float32)
    want_scale = np.zeros((t * k, 5), np.float32)
    for i in range(t):
        for s in range(k):
            if row[i, s] >= 0:
                want[row[i, s]] = x[i].float().cpu().numpy()
                if scale is not None:
                    want_scale[row[i, s]] = scale[i].cpu().numpy()
    assert p.rows.dtype == dtype and np.array_equal(p.rows.float().cpu().numpy(), want)
    assert np.array_equal(p.row_of_route.cpu().numpy(), row)
    assert np.array_equal(p.offsets.cpu().numpy(), offsets)
    if scale is not None:
        assert np.array_equal(p.scale.cpu().numpy(), want_scale)
    ops.permute.check_errors()


def plain_unpermute(rows, row, w):
    """64 bits: the sum and the sum of magnitudes."""
    row = row.long()
    held = (row >= 0)[..., None]
    y = torch.where(held, rows.double()[row.clamp_min(0)], 0.0) * w.double()[..., None]
    return y.sum(1), y.abs().sum(1)


SHAPES = [(1, 8, 384, 4096, 0.0), (64, 8, 384, 2048, 0.1), (37, 6, 64, 1001, 0.3), (300, 1, 8, 256, 0.0),
          (9, 17, 20, 130, 0.2), (1013, 6, 64, 512, 0.05), (4, 3, 5, 3, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,k,e,h,drop", SHAPES)
def test_unpermute_and_gradients(ops, dtype, t, k, e, h, drop):
    g = rng(7 * t + h)
    ids = routes(g, t, k, e, drop)
    row, _ = ops.permute.sort_routes(ids, e)
    rows = randn(g, t * k, h, dtype=dtype)
    dropped = row[row < 0].long()
    rows[~dropped] = float("nan")  # rows without an expert take no part
    w = torch.rand(t, k, generator=g, device="cuda")
    for out_dtype in {dtype, torch.float32}:
        r, wr = rows.clone().requires_grad_(), w.clone().requires_grad_()
        out = ops.permute.unpermute(r, row, wr, out_dtype=out_dtype)
        want, mag = plain_unpermute(rows, row, w)
        within(out, want, (k + 1) * 2.0**-23 * mag + U[out_dtype] * want.abs() + TINY[out_dtype])
        grad = randn(g, t, h, dtype=out_dtype)
        gr, gw = torch.autograd.grad(out, (r, wr), grad)
        held = (row >= 0)[..., None]
        back = torch.where(held, w.double()[..., None] * grad.double()[:, None], 0.0)
        want_gr = torch.empty(t * k, h, dtype=torch.float64, device="cuda")
        want_gr[torch.where(row < 0, ~row, row).long().view(-1)] = back.view(-1, h)
        within(gr, want_gr, 2 * U[dtype] * want_gr.abs() + TINY[dtype])
        prod = torch.where(held, rows.double()[row.long().clamp_min(0)], 0.0) * grad.double()[:, None]
        within(gw, prod.sum(-1), (h + 2) * 2.0**-23 * prod.abs().sum(-1))
    # without weights: plain sums
    out = ops.permute.unpermute(rows, row)
    want, mag = plain_unpermute(rows, row, torch.ones_like(w))
    within(out, want, (k + 1) * 2.0**-23 * mag + U[dtype] * want.abs() + TINY[dtype])
    ops.permute.check_errors()


@pytest.mark.gpu
def test_unpermute_gradients_one_at_a_time(ops):
    """Rows without weights, weights alone, and an expanded gradient (no row of its own in memory)."""
    g = rng(21)
    t, k, e, h = 23, 3, 7, 96
    row, _ = ops.permute.sort_routes(routes(g, t, k, e, 0.2), e)
    rows, w = randn(g, t * k, h), torch.rand(t, k, generator=g, device="cuda")
    r = rows.clone().requires_grad_()
    gr, = torch.autograd.grad(ops.permute.unpermute(r, row).sum(), r)
    want = torch.zeros(t * k, h, device="cuda")
    want[row[row >= 0].long()] = 1.0
    assert torch.equal(gr, want)
    wr = w.clone().requires_grad_()
    gw, = torch.autograd.grad(ops.permute.unpermute(rows, row, wr).sum(), wr)
    y = torch.where((row >= 0)[..., None], rows.double()[row.long().clamp_min(0)], 0.0)
    within(gw, y.sum(-1), (h + 2) * 2.0**-23 * y.abs().sum(-1))
    gr, gw = ops.permute.unpermute_grad(torch.ones(t, h, device="cuda"), rows, row, None)
    assert gw is None and torch.equal(gr, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k,e,h,drop", SHAPES)
def test_permute_gradient(ops, dtype, t, k, e, h, drop):
    g = rng(t + 11)
    ids = routes(g, t, k, e, drop)
    x = randn(g, t, h, dtype=dtype).requires_grad_()
    p = ops.permute.permute(x, ids, e)
    grad = randn(g, t * k, h, dtype=dtype)
    dropped = p.row_of_route[p.row_of_route < 0].long()
    grad[~dropped] = float("inf")  # a gradient of a row of zeros reaches no token
    gx, = torch.autograd.grad(p.rows, x, grad)
    want, mag = plain_unpermute(grad, p.row_of_route, torch.ones(t, k, device="cuda"))
    within(gx, want, (k + 1) * 2.0**-23 * mag + U[dtype] * want.abs() + TINY[dtype])


@pytest.mark.gpu
def test_gradients_against_differences(ops):
    """Both operators are linear in their rows: a central difference is exact but for f32 rounding."""
    g = rng(3)
    t, k, e, h = 12, 3, 5, 20
    ids = routes(g, t, k, e, 0.2)
    x, dx = randn(g, t, h), randn(g, t, h)
    w, dw = torch.rand(t, k, generator=g, device="cuda"), randn(g, t, k)
    c = randn(g, t, h)

    def f(x, w):
        p = ops.permute.permute(x, ids, e)
        return ops.permute.unpermute(p.rows * p.rows, p.row_of_route, w)

    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad((f(xr, wr) * c).sum(), (xr, wr))
    step = 2.0**-8  # f is quadratic in x: central differences have no truncation error
    num = ((f(x + step * dx, w).double() * c).sum() - (f(x - step * dx, w).double() * c).sum()) / (2 * step)
    mag = float((f(x.abs() + step * dx.abs(), w).double() * c.abs()).sum())
    assert abs(float(num) - float((gx.double() * dx).sum())) <= 16 * 2.0**-23 * mag / step
    num = ((f(x, w + step * dw).double() * c).sum() - (f(x, w - step * dw).double() * c).sum()) / (2 * step)
    assert abs(float(num) - float((gw.double() * dw).sum())) <= 16 * 2.0**-23 * mag * (1 + float(dw.abs().max())) / step


# ------------------------------------------------------------------- quantizer
def plain_quantize(x):
    """The definition in f32, step by step (numpy has no E4M3: torch's cast rounds to nearest even)."""
    rows, width = x.shape
    kb = -(-width // 128)
    b = torch.zeros(rows, kb * 128, device=x.device)
    b[:, :width] = x.float()
    b = b.view(rows, kb, 128)
    amax = b.abs().amax(-1).clamp_min(1e-30)
    top = torch.full_like(amax, 448.0)  # torch turns a quotient with a plain number into a product with its reciprocal
    q = (b * (top / amax)[..., None]).view(rows, -1)[:, :width]
    return q.to(E4M3), amax / top


def same_bits(a, b):
    """Equal E4M3 codes, every NaN alike."""
    assert torch.equal(a.float().nan_to_num(nan=1e9), b.float().nan_to_num(nan=1e9))


def dequantize(q, scale):
    return q.double() * scale.double().repeat_interleave(128, -1)[..., : q.shape[-1]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width,stride", [(1, 4096, 0), (3, 128, 0), (33, 1408, 0), (5, 1, 0), (17, 130, 0),
                                               (64, 2049, 0), (9, 256, 8), (9, 256, 5), (20000, 136, 0)])
def test_quantize_rows(ops, dtype, rows, width, stride):
    g = rng(rows + width)
    x = (randn(g, rows, width + stride) * torch.exp(3 * randn(g, rows, 1))).to(dtype)[:, :width]
    q, scale = ops.fp8.quantize(x)
    want_q, want_scale = plain_quantize(x)
    assert torch.equal(scale, want_scale)
    same_bits(q, want_q)


@pytest.mark.gpu
def test_quantize_special_values(ops):
    x = torch.zeros(8, 256, device="cuda")
    x[1, 3] = float("nan")
    x[2, 200] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = 1e-38
    x[5] = torch.finfo(torch.float32).max
    x[6, 5], x[6, 9] = 2.0**-140, -1e-31
    x[7, 128:] = -0.0
    q, scale = ops.fp8.quantize(x)
    want_q, want_scale = plain_quantize(x)
    assert torch.equal(scale.nan_to_num(nan=-1), want_scale.nan_to_num(nan=-1))
    same_bits(q[[0, 1, 4, 5, 6, 7]], want_q[[0, 1, 4, 5, 6, 7]])
    d = dequantize(q, scale)
    assert bool(d[1, :128].isnan().all()) and not bool(d[1, 128:].isnan().any())
    assert bool(d[2, 128:].isnan().all()) and bool(d[3, :128].isnan().all())
    assert float(d[0].abs().max()) == 0.0


def plain_swiglu(h, limit):
    gate, up = h.double().chunk(2, 1)
    g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
    return gate, up, g, u, torch.sigmoid(g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width,limit,stride", [(1, 2048, 10.0, 0), (37, 1408, 10.0, 0), (5, 129, 1.0, 0),
                                                     (300, 64, None, 0), (11, 72, 10.0, 8), (2, 1, 10.0, 1)])
def test_swiglu_quantize_and_gradient(ops, dtype, rows, width, limit, stride):
    g = rng(rows * width)
    h = (6 * randn(g, rows, 2 * width + stride)).to(dtype)[:, : 2 * width]
    lim = float("inf") if limit is None else limit
    gate, up, gg, u, s = plain_swiglu(h, lim)
    a = gg * s * u
    q, scale = ops.fp8.swiglu_quantize(h, limit=limit)
    amax = torch.zeros(rows, -(-width // 128) * 128, dtype=torch.float64, device="cuda")
    amax[:, :width] = a.abs()
    amax = amax.view(rows, -1, 128).amax(-1).clamp_min(1e-30)
    f32 = 8 * 2.0**-24  # exp, sum, quotient, product and the scale's own roundings
    within(scale, amax / 448, f32 * amax / 448)
    # half a step: 2^-4 of a normal value, 2^-10 of the scale below it
    wide = scale.double().repeat_interleave(128, 1)[:, :width]
    within(dequantize(q, scale), a, (2.0**-4 * a.abs() + 2.0**-10 * wide) * (1 + 2.0**-18) + f32 * 448 * wide)
    d = randn(g, rows, width, dtype=dtype)
    got = ops.fp8.swiglu_grad(h, d, limit=limit)
    dg = torch.where(gate > lim, 0.0, d.double() * u * (s + gg * s * (1 - s)))
    du = torch.where(up.abs() > lim, 0.0, d.double() * gg * s)
    want = torch.cat([dg, du], 1)
    # 1 - s and 1 + g (1 - s) cancel for large |g|: errors relative to the terms
    mag = torch.cat([d.double().abs() * u.abs() * (s + gg.abs() * s), d.double().abs() * gg.abs() * s], 1)
    within(got, want, U[dtype] * want.abs() + 16 * 2.0**-24 * mag + TINY[dtype])


@pytest.mark.gpu
def test_swiglu_gradient_against_differences(ops):
    g = rng(5)
    h = 4 * randn(g, 7, 2 * 40)
    d = randn(g, 7, 40)
    got = ops.fp8.swiglu_grad(h, d, limit=3.0).double()
    gate, up, *_ = plain_swiglu(h, 3.0)

    def f(v):
        _, _, gg, u, s = plain_swiglu(v, 3.0)
        return (gg * s * u * d.double()).sum()

    step = 1e-6
    for i, j in [(0, 0), (1, 13), (2, 39), (3, 40), (4, 57), (6, 79), (5, 20), (6, 61)]:
        near = gate[i, j % 40] if j < 40 else up[i, j - 40].abs()
        assert abs(float(near) - 3.0) > 1e-4  # not at the bound's corner
        v = h.double().clone()
        v[i, j] += step
        up_ = f(v)
        v[i, j] -= 2 * step
        num = float(up_ - f(v)) / (2 * step)
        assert abs(num - float(got[i, j])) <= 1e-5 * (1 + abs(num))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lead,n,k", [((), 128, 128), ((), 2816, 2048), ((), 300, 200), ((), 129, 17), ((3,), 200, 272),
                                      ((2,), 130, 129)])
def test_quantize_and_transpose_weights(ops, dtype, lead, n, k):
    g = rng(n + k)
    w = (0.02 * randn(g, *lead, n, k)).to(dtype)
    q, scale = ops.fp8.quantize_weight(w)
    nb, kb = -(-n // 128), -(-k // 128)
    pad = torch.zeros(*lead, nb * 128, kb * 128, device="cuda")
    pad[..., :n, :k] = w.float()
    blocks = pad.view(*lead, nb, 128, kb, 128)
    amax = blocks.abs().amax((-3, -1)).clamp_min(1e-30)
    top = torch.full_like(amax, 448.0)
    assert torch.equal(scale, amax / top)
    want = (blocks * (top / amax)[..., :, None, :, None]).view(*lead, nb * 128, kb * 128)[..., :n, :k].to(E4M3)
    same_bits(q, want)
    qt, st = ops.fp8.transpose_weight(q, scale)
    assert torch.equal(qt.view(torch.uint8), q.view(torch.uint8).transpose(-1, -2).contiguous())
    assert torch.equal(st, scale.transpose(-1, -2).contiguous())


# -------------------------------------------------------------------- products
def weights(g, *shape):
    """E4M3 weights with a scale per 128 x 128 block, of any scale."""
    q = (60 * randn(g, *shape)).clamp(-448, 448).to(E4M3)
    lead, (n, k) = shape[:-2], shape[-2:]
    return q, torch.rand(*lead, -(-n // 128), -(-k // 128), generator=g, device="cuda") * 1e-3 + 1e-4


def plain_product(q, scale, w, w_scale):
    """64 bits: the product and the product of magnitudes."""
    a = dequantize(q, scale)
    b = dequantize(w, w_scale.repeat_interleave(128, -2)[..., : w.shape[-2], :])
    return a @ b.T, a.abs() @ b.abs().T


def sum_bound(mag, k):
    """128 products a block, a scale's two roundings and one addition per block, each losing up to 2^-23."""
    return (128 + -(-k // 128) + 4) * 2.0**-23 * mag


PRODUCTS = [(1, 4096, 4096), (1, 16, 16), (2, 130, 144), (8, 2816, 2048), (9, 2048, 1408), (16, 257, 256),
            (17, 384, 128), (64, 512, 4096), (127, 129, 112), (128, 128, 128), (129, 640, 1424), (333, 2816, 2048),
            (1000, 2049, 272), (3000, 4096, 512), (5, 33, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_matmul(ops, m, n, k, out_dtype):
    g = rng(m + n + k)
    q, scale = ops.fp8.quantize(randn(g, m, k))
    w, w_scale = weights(g, n, k)
    got = ops.fp8.matmul(q, scale, w, w_scale, out_dtype=out_dtype)
    want, mag = plain_product(q, scale, w, w_scale)
    within(got, want, sum_bound(mag, k) + U[out_dtype] * want.abs() + TINY[out_dtype])
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,stride", [(1, 4096, 4096, 0), (1, 48, 144, 0), (3, 2816, 2048, 8), (8, 256, 1408, 0),
                                          (8, 256, 1408, 3), (9, 256, 1408, 0), (70, 320, 512, 16)])
def test_linear_and_gradient(ops, dtype, m, n, k, stride):
    g = rng(m * n)
    x = randn(g, m, k + stride, dtype=dtype)[:, :k]
    w, w_scale = weights(g, n, k)
    q, scale = plain_quantize(x)
    want, mag = plain_product(q, scale, w, w_scale)
    got = ops.fp8.linear(x, w, w_scale)
    assert got.dtype == dtype
    within(got, want, sum_bound(mag, k) + U[dtype] * want.abs() + TINY[dtype])
    grad = randn(g, m, n, dtype=dtype)
    wt, wt_scale = w.view(torch.uint8).t().contiguous().view(E4M3), w_scale.t().contiguous()
    gq, gs = plain_quantize(grad)
    want, mag = plain_product(gq, gs, wt, wt_scale)
    for kept in ((), (wt, wt_scale)):
        xr = x.detach().requires_grad_()
        gx, = torch.autograd.grad(ops.fp8.linear(xr, w, w_scale, *kept), xr, grad)
        within(gx, want, sum_bound(mag, n) + U[dtype] * want.abs() + TINY[dtype])


@pytest.mark.gpu
def test_linear_gradient_against_differences(ops):
    """The product without its quantizer is linear in the rows: with every value of x and of the gradient exact
    in E4M3 and every block's largest 448, the difference of two calls is the gradient's."""
    g = rng(17)
    m, n, k = 40, 48, 64
    w, w_scale = weights(g, n, k)

    def grid(*shape):
        v = torch.randint(-15, 16, shape, generator=g, device="cuda").float()
        v[:, 0] = 448.0
        return v

    x, c = grid(m, k), grid(m, n)
    xr = x.clone().requires_grad_()
    gx, = torch.autograd.grad(ops.fp8.linear(xr, w, w_scale), xr, c)
    dx = torch.zeros(m, k, device="cuda")
    dx[:, 1:] = torch.randint(-1, 2, (m, k - 1), generator=g, device="cuda").float()
    num = ((ops.fp8.linear(x + dx, w, w_scale).double() - ops.fp8.linear(x - dx, w, w_scale).double()) * c).sum(1) / 2
    _, mag = plain_product(*plain_quantize(x.abs() + 1), w, w_scale)
    bound = 2 * (sum_bound(mag, k) * c.abs()).sum(1) + sum_bound(1, n) * 64 * (gx.double().abs()).sum(1)
    _, mag_g = plain_product(*plain_quantize(c.abs()), w.view(torch.uint8).t().contiguous().view(E4M3),
                             w_scale.t().contiguous())
    bound = bound + sum_bound(mag_g, n).sum(1)
    assert bool(((num - (gx.double() * dx).sum(1)).abs() <= bound).all())


def offsets_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


GROUPED = [
    ([1], 0, 64, 128), ([0, 0, 1, 0], 0, 130, 144), ([3, 0, 1, 9, 0, 2], 4, 256, 512), ([0, 0], 5, 64, 64),
    ([8, 16, 7, 17], 0, 2816, 256), ([200, 0, 1, 129, 128, 3], 1, 384, 1424), ([1000, 1], 0, 129, 272),
    ([2] * 64, 0, 512, 4096), ([1, 0, 2] * 100, 10, 144, 2048), ([40, 0, 300] * 10, 7, 272, 384),
    ([12] * 20, 0, 96, 1408), ([0] * 1023 + [5], 0, 32, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,tail,n,k", GROUPED)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_grouped_matmul(ops, counts, tail, n, k, out_dtype):
    g = rng(n + k + len(counts))
    off = offsets_of(counts)
    s = int(off[-1]) + tail
    q, scale = ops.fp8.quantize(randn(g, s, k))
    w, w_scale = weights(g, len(counts), n, k)
    if tail:  # rows without an expert are not read into any sum
        q.view(torch.uint8)[int(off[-1]):] = 0x7F
    got = ops.fp8.grouped_matmul(q, scale, off, w, w_scale, out_dtype=out_dtype)
    for e, c in enumerate(counts):
        if c:
            rows = slice(int(off[e]), int(off[e + 1]))
            want, mag = plain_product(q[rows], scale[rows], w[e], w_scale[e])
            within(got[rows], want, sum_bound(mag, k) + U[out_dtype] * want.abs() + TINY[out_dtype])
    assert float(got[int(off[-1]):].abs().sum()) == 0.0
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 12, 40, 300])
def test_nan_stays_in_its_row(ops, m):
    g = rng(m)
    x = randn(g, m, 512, dtype=torch.bfloat16)
    w, w_scale = weights(g, 256, 512)
    clean = ops.fp8.linear(x, w, w_scale)
    x[m // 2, 300] = float("nan")
    got = ops.fp8.linear(x, w, w_scale)
    assert bool(got[m // 2].isnan().all())
    keep = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_bad_offsets_and_rows_are_reported(ops):
    """Values the kernels check themselves: nothing out of range is touched, check_errors raises once."""
    from b200moe._lib import B200MoeError

    g = rng(1)
    w, w_scale = weights(g, 2, 64, 128)
    for s in (4, 200):
        q, scale = ops.fp8.quantize(randn(g, s, 128))
        bad = torch.tensor([0, s + 7, s], dtype=torch.int32, device="cuda")
        ops.fp8.grouped_matmul(q, scale, bad, w, w_scale)
        with pytest.raises(B200MoeError):
            ops.fp8.check_errors()
        ops.fp8.check_errors()
    row = torch.tensor([[0, 99]], dtype=torch.int32, device="cuda")
    out = ops.permute.unpermute(torch.ones(2, 8, device="cuda"), row)
    assert torch.equal(out, torch.ones(1, 8, device="cuda"))
    with pytest.raises(B200MoeError):
        ops.permute.check_errors()


@pytest.mark.gpu
def test_empty_batches(ops):
    dev = "cuda"
    ids = torch.empty(0, 4, dtype=torch.int32, device=dev)
    p = ops.permute.permute(torch.empty(0, 64, device=dev), ids, 8)
    assert p.rows.shape == (0, 64) and p.offsets.tolist() == [0] * 9
    assert ops.permute.unpermute(p.rows, p.row_of_route).shape == (0, 64)
    q, scale = ops.fp8.quantize(torch.empty(0, 64, device=dev))
    g = rng(0)
    w, ws = weights(g, 8, 32, 64)
    assert ops.fp8.grouped_matmul(q, scale, p.offsets, w, ws).shape == (0, 32)
    assert ops.fp8.linear(torch.empty(0, 64, device=dev), w[0], ws[0]).shape == (0, 32)


@pytest.mark.gpu
def test_gradients_refuse_a_second_differentiation(ops):
    """A gradient of a gradient is refused, not left out."""
    g = rng(2)
    ids = routes(g, 5, 2, 4)
    x = randn(g, 5, 32).requires_grad_()
    w, ws = weights(g, 48, 32)
    p = ops.permute.permute(x, ids, 4)
    for y in (p.rows, ops.permute.unpermute(p.rows, p.row_of_route), ops.fp8.linear(x, w, ws)):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y.sum(), x, create_graph=True, retain_graph=True)


@pytest.mark.gpu
def test_offsets_past_32_bits(ops):
    """2.4 million rows of 1024: elements past 2^31 in every operator; the last rows are looked at."""
    g = rng(31)
    t, k, e, h = 300_000, 8, 16, 1024
    ids = torch.randint(0, e, (t, k), generator=g, device="cuda", dtype=torch.int32)
    x = randn(g, t, h, dtype=torch.bfloat16)
    p = ops.permute.permute(x, ids, e)
    assert p.rows.numel() > 2**31
    tail = p.row_of_route[-500:].long()
    assert torch.equal(p.rows[tail], x[-500:, None].expand(-1, k, -1))
    w = torch.rand(t, k, generator=g, device="cuda")
    out = ops.permute.unpermute(p.rows, p.row_of_route, w)[-500:]
    want, mag = plain_unpermute(p.rows[tail].reshape(-1, h), torch.arange(500 * k, device="cuda").view(500, k), w[-500:])
    within(out, want, (k + 1) * 2.0**-23 * mag + U[torch.bfloat16] * want.abs() + TINY[torch.bfloat16])
    grad_rows, _ = ops.permute.unpermute_grad(x, p.rows, p.row_of_route, w, need_weights=False)
    back = w[-500:, :, None].double() * x[-500:, None].double()
    within(grad_rows[tail], back, 2 * U[torch.bfloat16] * back.abs() + TINY[torch.bfloat16])
    del grad_rows
    q, scale = ops.fp8.quantize(p.rows)
    want_q, want_scale = plain_quantize(p.rows[-300:])
    assert torch.equal(scale[-300:], want_scale)
    same_bits(q[-300:], want_q)
    wq, ws = weights(g, e, h, h)
    y = ops.fp8.grouped_matmul(q, scale, p.offsets, wq, ws)[-300:]  # the last expert's
    want, mag = plain_product(q[-300:], scale[-300:], wq[-1], ws[-1])
    within(y, want, sum_bound(mag, h) + U[torch.bfloat16] * want.abs() + TINY[torch.bfloat16])
    del y, q, scale
    half = p.rows.view(t * k // 2, 2 * h)
    a, a_scale = ops.fp8.swiglu_quantize(half)
    a0, s0 = ops.fp8.swiglu_quantize(half[-100:])
    same_bits(a[-100:], a0)
    assert torch.equal(a_scale[-100:], s0)
    d = ops.fp8.swiglu_grad(half, half[:, :h])
    assert torch.equal(d[-100:], ops.fp8.swiglu_grad(half[-100:], half[-100:, :h]))


@pytest.mark.gpu
def test_same_bits_and_another_stream(ops):
    g = rng(9)
    t, k, e, h, i = 50, 4, 16, 256, 128
    m = ops.experts.Fp8Experts.from_weights(0.05 * randn(g, e, 2 * i, h), 0.05 * randn(g, e, h, i))
    x, ids = randn(g, t, h, dtype=torch.bfloat16), routes(g, t, k, e, 0.1)
    w = torch.rand(t, k, generator=g, device="cuda")
    want = m(x, ids, w)
    assert torch.equal(want, m(x, ids, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m(x, ids, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m(x, ids, w)
    x.copy_(randn(g, t, h, dtype=torch.bfloat16))
    graph.replay()
    assert torch.equal(got, m(x, ids, w))


# ---------------------------------------------------------------- the whole path
def rounded(v, dtype):
    return v.to(dtype).double()


def requantized(v):
    """What the quantizer makes of values that are exact in f32."""
    return dequantize(*plain_quantize(v.float()))


def plain_experts(x, ids, w, q13, q2, limit, grad):
    """The path and its gradients expert by expert in 64 bits, rounded where the framework's path stores 16 or 8
    bits: (out, grad x, grad w)."""
    dt = x.dtype
    xq = requantized(x)
    out, gx = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros_like(x, dtype=torch.float64)
    gw = torch.zeros_like(w, dtype=torch.float64)
    for e in range(q13.shape[0]):
        t, s = torch.nonzero(ids == e, as_tuple=True)
        if len(t) == 0:
            continue
        h = rounded(xq[t] @ q13[e].T, dt)
        gate, up, g, u, sig = plain_swiglu(h, limit)
        y = rounded(requantized(g * sig * u) @ q2[e].T, dt)
        we = w[t, s, None].double()
        out.index_add_(0, t, we * y)
        ge = grad[t].double()
        gw[t, s] = (ge * y).sum(1)
        ga = rounded(requantized(rounded(we * ge, dt)) @ q2[e], dt)
        dg = torch.where(gate > limit, 0.0, ga * u * (sig + g * sig * (1 - sig)))
        du = torch.where(up.abs() > limit, 0.0, ga * g * sig)
        gx.index_add_(0, t, rounded(requantized(rounded(torch.cat([dg, du], 1), dt)) @ q13[e], dt))
    return out, gx, gw


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,e,h,i", [(1, 4, 16, 512, 256), (70, 6, 16, 512, 352), (900, 4, 8, 256, 128)])
def test_fp8_experts(ops, t, k, e, h, i):
    """In the norm within twice the last rounding, 2 * 2^-8: one share for that rounding itself, one for values
    whose 32-bit sum falls on the other side of an earlier rounding's boundary than the 64-bit one (a share of
    about 2^-20 / 2^-8 of the values, each one step of at most 2^-3 off)."""
    g = rng(t)
    w13, w2 = 0.05 * randn(g, e, 2 * i, h), 0.05 * randn(g, e, h, i)
    m = ops.experts.Fp8Experts.from_weights(w13, w2, trainable=True)
    x, ids = randn(g, t, h, dtype=torch.bfloat16), routes(g, t, k, e, 0.1)
    w = torch.rand(t, k, generator=g, device="cuda")
    grad = randn(g, t, h, dtype=torch.bfloat16)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = m(xr, ids, wr)
    gx, gw = torch.autograd.grad(out, (xr, wr), grad)
    assert torch.equal(out, m(x, ids, w)) and out.dtype == x.dtype
    wide = lambda q, s: dequantize(q, s.repeat_interleave(128, -2)[..., : q.shape[-2], :])  # noqa: E731
    want, want_gx, want_gw = plain_experts(x, ids, w, wide(m.w13, m.w13_scale), wide(m.w2, m.w2_scale), 10.0, grad)
    for got, ref in ((out, want), (gx, want_gx), (gw, want_gw)):
        assert float((got.detach().double() - ref).norm()) <= 2 * 2.0**-8 * float(ref.norm())
    assert float(gw[ids < 0].abs().sum()) == 0.0
    ops.fp8.check_errors()


# -------------------------------------------------------------------- refusals
def test_refusals_on_host_tensors(pkg):
    """Every public call refuses what is not a CUDA tensor, before it looks at anything else."""
    from b200moe import experts, fp8, permute

    x, ids = torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.int32)
    q, s = torch.zeros(2, 16).to(E4M3), torch.zeros(2, 1)
    w, ws = torch.zeros(16, 16).to(E4M3), torch.zeros(1, 1)
    calls = [lambda: permute.permute(x, ids, 4), lambda: permute.unpermute(x, ids),
             lambda: permute.unpermute_grad(x, x, ids, None), lambda: permute.sort_routes(ids, 4),
             lambda: fp8.quantize(x), lambda: fp8.swiglu_quantize(x), lambda: fp8.swiglu_grad(x, x[:, :8]),
             lambda: fp8.quantize_weight(x), lambda: fp8.transpose_weight(w, ws), lambda: fp8.matmul(q, s, w, ws),
             lambda: fp8.grouped_matmul(q, s, ids[0], w[None], ws[None]), lambda: fp8.linear(x, w, ws),
             lambda: experts.Fp8Experts(w[None], ws[None], w[None], ws[None])]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_refusals(ops):
    P, F = ops.permute, ops.fp8
    g = rng(0)
    dev = "cuda"
    x = randn(g, 6, 64)
    ids = torch.zeros(6, 2, dtype=torch.int32, device=dev)
    rows, row = randn(g, 12, 64), torch.zeros(6, 2, dtype=torch.int32, device=dev)
    q, s = F.quantize(x)
    w, ws = weights(g, 32, 64)
    we, wse = weights(g, 2, 32, 64)
    off = offsets_of([2, 4])
    bad = [
        lambda: P.permute(x.double(), ids, 4), lambda: P.permute(x, ids.long(), 4), lambda: P.permute(x, ids[:5], 4),
        lambda: P.permute(x, ids, 0), lambda: P.permute(x, ids, 1025), lambda: P.permute(x.t(), ids, 4),
        lambda: P.permute(x[:, ::2], ids, 4), lambda: P.permute(x, ids, 4, scale=s[:5]),
        lambda: P.permute(x.clone().requires_grad_(), ids, 4, scale=s),
        lambda: P.unpermute(rows[:11], row), lambda: P.unpermute(rows, row.long()),
        lambda: P.unpermute(rows, row, torch.ones(6, 3, device=dev)), lambda: P.unpermute(rows[:, :32], row),
        lambda: P.unpermute(rows, row, torch.ones(6, 2, device=dev, dtype=torch.bfloat16)),
        lambda: P.unpermute(rows, row, out_dtype=torch.bfloat16), lambda: P.unpermute(rows.to(E4M3), row),
        lambda: F.quantize(x.double()), lambda: F.quantize(x[0]), lambda: F.quantize(x[:, :0]),
        lambda: F.swiglu_quantize(x[:, :63]), lambda: F.swiglu_quantize(x, limit=0.0),
        lambda: F.swiglu_quantize(x, limit=float("nan")), lambda: F.swiglu_grad(x, x), lambda: F.swiglu_grad(x, x[:, :32].half()),
        lambda: F.matmul(q, s[:, :0], w, ws), lambda: F.matmul(q, s, w[:, :32], ws), lambda: F.matmul(q, s, w, ws[0]),
        lambda: F.matmul(q[:, :24], s, w[:, :24].contiguous(), ws), lambda: F.matmul(x, s, w, ws),
        lambda: F.matmul(q[:, :24].contiguous(), s, w[:, :24].contiguous(), ws),  # K not a multiple of 16
        lambda: F.matmul(q, s, w, ws, out_dtype=torch.int32), lambda: F.matmul(q.view(torch.uint8), s, w, ws),
        lambda: F.matmul(q.view(torch.float8_e5m2), s, w, ws),
        lambda: F.grouped_matmul(q, s, off[:2], we, wse), lambda: F.grouped_matmul(q, s, off.long(), we, wse),
        lambda: F.grouped_matmul(q, s, off, w, ws), lambda: F.linear(x, w, ws, wt=w),
        lambda: F.linear(x, w, ws, w, ws),  # not the transposed shape
        lambda: F.linear(x.clone().requires_grad_(), w[:31], ws),  # the gradient's K
        lambda: F.quantize_weight(x[0]), lambda: F.quantize_weight(x[:, :0]),
        lambda: ops.experts.Fp8Experts(we, wse, we, wse),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    m = ops.experts.Fp8Experts.from_weights(randn(g, 2, 64, 64), randn(g, 2, 64, 32))
    for args in [(x, ids, torch.ones(6, 2, device=dev)), (x.half()[:, :32], ids, torch.ones(6, 2, device=dev)),
                 (x.half(), ids, torch.ones(6, 3, device=dev)),
                 (x.half().requires_grad_(), ids, torch.ones(6, 2, device=dev))]:
        with pytest.raises(ValueError):
            m(*args)
    # an address off the 16 bytes that the copies need is refused by the library
    from b200moe._lib import B200MoeError

    flat = torch.zeros(12 * 64 + 16, dtype=torch.uint8, device=dev).view(E4M3)
    with pytest.raises(B200MoeError):
        F.matmul(flat[8: 8 + 6 * 64].view(6, 64), s, w, ws)


@pytest.mark.gpu
def test_example_learns_and_serves():
    """The example's loss falls, and single tokens give the batch's rows up to the last rounding (both differ from the
    exact sum by half a bf16 step, 2^-9 in the rms at most)."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "fp8_experts.py"
    spec = importlib.util.spec_from_file_location("fp8_experts_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    got = mod.main(["--tokens", "96", "--hidden", "256", "--inter", "128", "--experts", "8", "--steps", "20"])
    assert got["last"] < 0.9 * got["first"]
    assert got["single"] <= 2 * 2.0**-8
