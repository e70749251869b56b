"""The root-mean-square norm (``norm``) and its gradient against 64-bit forms.

Tolerances.  A thread adds 16 squares and up to 4 such sums, a warp 5, a CTA 8: at most 53 roundings of 2^-24 in the mean,
half of that in the root, 6 more operations to y: y is off by less than 2^-19 of itself before its own rounding.  A
gradient adds the mean of g u, off by 2^-18 of the mean of magnitudes; the weight's adds one rounding per row."""

from __future__ import annotations

import pytest
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-149}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6
SIZES = [(1, 1), (1, 4096), (3, 7), (9, 32), (64, 512), (17, 513), (33, 520), (300, 1401), (5, 2048), (1013, 2056),
         (2, 8192), (2, 8193), (3, 12296), (2, 16384), (2, 16383)]


@pytest.fixture(scope="module")
def ops(pkg):
    from b200moe import fp4, fp8, norm

    return type("Ops", (), {"fp4": fp4, "fp8": fp8, "norm": norm})


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def within(got, want, bound):
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), f"worst excess {float((d - bound).max()):.3e}"


def formula(s, w, eps=EPS):
    s = s.double()
    rstd = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    return s * rstd * w.double(), rstd


def inputs(m, h, dtype, res, weight_f32, pad=0):
    x = randn(m + h, m, h + pad, dtype=dtype)[:, :h]
    r = None if res == "none" else (randn(h, m, h + pad) * 3).to(torch.float32 if res == "f32" else dtype)[:, :h]
    w = (1 + 0.3 * randn(m, h)).to(torch.float32 if weight_f32 else dtype)
    return x, r, w


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("res,weight_f32", [("none", False), ("same", True), ("f32", False)])
@pytest.mark.parametrize("m,h", SIZES)
def test_norm(ops, dtype, res, weight_f32, m, h):
    for pad in (0, 8, 1):
        x, r, w = inputs(m, h, dtype, res, weight_f32, pad)
        y, total = ops.norm.rms_norm(x, w, r, EPS)
        if r is None:
            assert total is None
            s = x
        else:
            assert total.dtype == r.dtype
            assert torch.equal(total, (x.float() + r.float()).to(r.dtype))
            s = total
        want, _ = formula(s, w)
        assert y.dtype == dtype
        within(y, want, want.abs() * (2.0**-19 + U[dtype]) + TINY[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("res,weight_f32", [("none", True), ("same", False), ("f32", True)])
@pytest.mark.parametrize("m,h", [(1, 1), (1, 4096), (3, 7), (9, 32), (64, 512), (17, 513), (2500, 96), (300, 1401),
                                 (1013, 2056), (900, 4096), (3, 12296), (2, 16383)])
def test_gradients(ops, dtype, res, weight_f32, m, h):
    x, r, w = inputs(m, h, dtype, res, weight_f32)
    leaves = [t.clone().requires_grad_() for t in (x, w)] + ([] if r is None else [r.clone().requires_grad_()])
    y, total = ops.norm.rms_norm(leaves[0], leaves[1], None if r is None else leaves[2], EPS)
    dy = randn(1, m, h, dtype=dtype)
    outs, grads = [y], [dy]
    if r is not None:
        outs.append(total)
        grads.append(randn(2, m, h, dtype=r.dtype))
    got = torch.autograd.grad(outs, leaves, grads)
    s = x if r is None else total.detach()
    _, rstd = formula(s, w)
    u, g = s.double() * rstd, dy.double() * w.double()
    mean, size = (g * u).mean(1, keepdim=True), (g * u).abs().mean(1, keepdim=True)
    ds = rstd * (g - u * mean)
    bound = rstd * (g.abs() + u.abs() * size) * 2.0**-18
    if r is not None:
        ds = ds + grads[1].double()
        bound = bound + ds.abs() * 2.0**-23
        within(got[2], ds, bound + ds.abs() * U[r.dtype] + TINY[r.dtype])
        assert got[2].dtype == r.dtype
    within(got[0], ds, bound + ds.abs() * U[dtype] + TINY[dtype])
    dw, mag = (dy.double() * u).sum(0), (dy.double() * u).abs().sum(0)
    within(got[1], dw, mag * ((m + 64) * 2.0**-24 + 2.0**-19) + dw.abs() * U[w.dtype] + TINY[w.dtype])
    again = torch.autograd.grad(ops.norm.rms_norm(leaves[0], leaves[1], None if r is None else leaves[2], EPS)[: len(outs)],
                                leaves, grads)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.gpu
def test_gradient_against_differences(ops):
    """f32: central differences of a sum of both outputs along random directions; their own error is of the step's
    square times the third derivative (step 2^-6, values near 1: 1e-3) and 2^-24 of the sum over the step (4e-4)."""
    x, r, w = inputs(7, 40, torch.float32, "same", True)
    cy, cs = randn(5, 7, 40).double(), randn(6, 7, 40).double()

    def value(x, r, w):
        y, total = ops.norm.rms_norm(x, w, r, EPS)
        return (y.double() * cy).sum() + (total.double() * cs).sum()

    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    grads = torch.autograd.grad(value(*leaves), leaves)
    for i in range(3):
        v = randn(9 + i, *leaves[i].shape)
        v /= v.norm()
        at = [[t + (0.0 if j != i else sign * 2.0**-6 * v) for j, t in enumerate((x, r, w))] for sign in (1, -1)]
        slope = float(value(*at[0]) - value(*at[1])) * 2.0**5
        assert abs(slope - float((grads[i] * v).sum())) < 2e-3 * max(1.0, abs(slope))


@pytest.mark.gpu
def test_gradients_that_are_not_all_asked_for(ops):
    x, r, w = inputs(30, 264, torch.bfloat16, "f32", False)
    dy, dt = randn(1, 30, 264, dtype=torch.bfloat16), randn(2, 30, 264)
    full = ops.norm.rms_norm_grad((x.float() + r), dy, w, dt)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0)):
        got = ops.norm.rms_norm_grad((x.float() + r), dy, w, dt, EPS, *map(bool, need))
        for g, f, n in zip(got, full, need):
            assert (g is None) if not n else torch.equal(g, f)
    # one output unused, an expanded gradient, a frozen weight
    a, b = x.clone().requires_grad_(), r.clone().requires_grad_()
    y, total = ops.norm.rms_norm(a, w, b)
    ga, gb = torch.autograd.grad(y.float().sum(), (a, b), retain_graph=True)
    zero = ops.norm.rms_norm_grad(total.detach(), torch.ones_like(y), w, None)
    assert torch.equal(ga, zero[0]) and torch.equal(gb, zero[1])
    ga, gb = torch.autograd.grad(total, (a, b), dt)
    assert torch.equal(gb, dt) and torch.equal(ga, dt.bfloat16())
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(ops.norm.rms_norm(a, w, b).y.sum(), a, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp8", "nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("res", ["none", "same", "f32"])
@pytest.mark.parametrize("m,h", [(1, 32), (1, 4096), (7, 96), (40, 512), (65, 544), (333, 2048), (9, 8192), (5, 8224),
                                 (2, 16384)])
def test_quantized_rows_are_those_of_the_norm(ops, fmt, dtype, res, m, h):
    """The quantizer's bits for y before its rounding, which the f32 norm of the stored sum returns."""
    for pad in (0, 3):
        x, r, w = inputs(m, h, dtype, res, False, pad)
        q, total, y = ops.norm.rms_norm_quantize(x, w, r, EPS, fmt, keep=True)
        plain = ops.norm.rms_norm(x, w, r, EPS)
        assert torch.equal(y, plain.y) and (total is None if r is None else torch.equal(total, plain.sum))
        s = x if r is None else total
        wide = ops.norm.rms_norm(s.float().contiguous(), w.float(), eps=EPS).y
        if fmt == "fp8":
            want, scale = ops.fp8.quantize(wide)
            assert torch.equal(q[0].view(torch.uint8), want.view(torch.uint8)) and torch.equal(q[1], scale)
        else:
            assert torch.equal(q.record, ops.fp4.quantize(wide, fmt).record) and q.columns == h
        none = ops.norm.rms_norm_quantize(x, w, r, EPS, fmt)
        assert none.y is None


@pytest.mark.gpu
@pytest.mark.parametrize("m,h", [(3, 1), (40, 1401), (2, 16383), (300, 130)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_fp8_rows_of_odd_width(ops, dtype, m, h):
    x, r, w = inputs(m, h, dtype, "same", True)
    (q, scale), total, _ = ops.norm.rms_norm_quantize(x, w, r, EPS)
    want, want_scale = ops.fp8.quantize(ops.norm.rms_norm(total.float(), w.float(), eps=EPS).y)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scale, want_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("h", [64, 2048, 1401])
def test_values_whose_squares_pass_f32(ops, h):
    """Rows near the type's ends: large ones are scaled before their squares, small ones are below eps."""
    base = randn(h, 6, h)
    x = base * torch.tensor([1e30, 3e37, 1e19, 1e-30, 0.0, 1.0], device="cuda")[:, None]
    w, dy = 1 + 0.1 * randn(1, h), randn(2, 6, h)
    y, _ = ops.norm.rms_norm(x, w)
    want, rstd = formula(x, w)
    within(y, want, want.abs() * 2.0**-18 + TINY[torch.float32])
    gx, _, gw = ops.norm.rms_norm_grad(x, dy, w)
    u, g = x.double() * rstd, dy.double() * w.double()
    ds = rstd * (g - u * (g * u).mean(1, keepdim=True))
    bound = rstd * (g.abs() + u.abs() * (g * u).abs().mean(1, keepdim=True)) * 2.0**-18
    within(gx, ds, bound + 4 * TINY[torch.float32] + bound * 2.0**-3 * 0)
    within(gw, (dy.double() * u).sum(0), (dy.double() * u).abs().sum(0) * 2.0**-18)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_value_that_is_no_number_stays_in_its_row(ops, bad):
    x, r, w = inputs(9, 256, torch.bfloat16, "same", False)
    x[4, 7] = bad
    good = [i for i in range(9) if i != 4]
    y, _ = ops.norm.rms_norm(x, w, r)
    assert y[4].isnan().any() and not y[good].isnan().any()
    for fmt in ("fp8", "nvfp4", "mxfp4"):
        q, _, _ = ops.norm.rms_norm_quantize(x, w, r, format=fmt)
        v = q[0].float() if fmt == "fp8" else ops.fp4.dequantize(q)
        assert v[4].isnan().any() and not v[good].isnan().any()


@pytest.mark.gpu
def test_empty_and_refused(ops):
    n = ops.norm
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16)
    assert n.rms_norm(x, w).y.shape == (0, 64) and n.rms_norm_quantize(x, w, x).rows[0].shape == (0, 64)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    ga, gb = torch.autograd.grad(n.rms_norm(a, b).y, (a, b), x)
    assert ga.shape == (0, 64) and not gb.any()
    x = randn(1, 8, 64, dtype=torch.bfloat16)
    for bad in (lambda: n.rms_norm(x, w[:32]), lambda: n.rms_norm(x, w.half()), lambda: n.rms_norm(x, w, x[:4]),
                lambda: n.rms_norm(x, w, x.half()), lambda: n.rms_norm(x, w, eps=0.0), lambda: n.rms_norm(x, w, eps=-1.0),
                lambda: n.rms_norm(x, w, eps=float("nan")), lambda: n.rms_norm(x.cpu(), w), lambda: n.rms_norm(x[0], w),
                lambda: n.rms_norm(x[:, ::2], w[::2].contiguous()), lambda: n.rms_norm(x, w, x[:1].expand(8, 64)),
                lambda: n.rms_norm(torch.zeros(2, 16385, device="cuda"), torch.ones(16385, device="cuda")),
                lambda: n.rms_norm_quantize(x, w, format="fp4"), lambda: n.rms_norm_quantize(x.clone().requires_grad_(), w),
                lambda: n.rms_norm_quantize(randn(1, 4, 40), torch.ones(40, device="cuda"), format="nvfp4"),
                lambda: n.rms_norm_grad(x, x.half(), w), lambda: n.rms_norm_grad(x, x, w, x.float())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_past_32_bit_offsets(ops):
    """More than 2^31 values: the last rows as by a call of their own, the weight's gradient as of the rows that count."""
    m, h = 540_001, 4096
    x, r = torch.zeros(m, h, device="cuda", dtype=torch.bfloat16), torch.zeros(m, h, device="cuda", dtype=torch.bfloat16)
    tail = slice(m - 40, m)
    x[tail], r[tail] = randn(1, 40, h), randn(2, 40, h)
    w = 1 + 0.1 * randn(3, h)
    y, total = ops.norm.rms_norm(x, w, r)
    want = ops.norm.rms_norm(x[tail], w, r[tail])
    assert torch.equal(y[tail], want.y) and torch.equal(total[tail], want.sum) and not y[:-40].any()
    q = ops.norm.rms_norm_quantize(x, w, r, format="nvfp4").rows.record
    assert torch.equal(q[tail], ops.norm.rms_norm_quantize(x[tail], w, r[tail], format="nvfp4").rows.record)
    del q, y
    gx, _, gw = ops.norm.rms_norm_grad(total, x, w, r)
    wx, _, ww = ops.norm.rms_norm_grad(total[tail], x[tail], w, r[tail])
    assert torch.equal(gx[tail], wx)
    _, rstd = formula(total[tail], w)
    mag = (x[tail].double() * total[tail].double() * rstd).abs().sum(0)
    within(gw, ww.double(), mag * 2.0**-18)


@pytest.mark.gpu
def test_leaves_get_gradients_of_their_own(ops):
    x, r, w = (t.requires_grad_() for t in inputs(6, 64, torch.bfloat16, "same", False))
    y, total = ops.norm.rms_norm(x, w, r)
    (y.float().sum() + total.float().sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    both = x.detach().clone().requires_grad_()  # the same tensor twice
    ops.norm.rms_norm(both, w, both).sum.float().sum().backward()
    assert torch.equal(both.grad, torch.full_like(both, 2.0))


@pytest.mark.gpu
def test_graph_replay(ops):
    x, r, w = inputs(130, 2048, torch.bfloat16, "same", False)
    g = torch.cuda.CUDAGraph()
    dy = randn(3, 130, 2048, dtype=torch.bfloat16)
    with torch.cuda.graph(g):
        y, total = ops.norm.rms_norm(x, w, r)
        grads = ops.norm.rms_norm_grad(total, dy, w)
        q = ops.norm.rms_norm_quantize(x, w, r, format="nvfp4")
    x.copy_(randn(4, 130, 2048, dtype=torch.bfloat16))
    g.replay()
    want = ops.norm.rms_norm(x, w, r)
    assert torch.equal(y, want.y) and torch.equal(total, want.sum)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.norm.rms_norm_grad(want.sum, dy, w)))
    assert torch.equal(q.rows.record, ops.norm.rms_norm_quantize(x, w, r, format="nvfp4").rows.record)
