"""Edges of the FP8 expert path's operators: extreme values, ranges, refusals and the sizes where one kernel gives way
to the next.  Expected values are plain torch forms in 64 bits, or in f32 step by step where the definition fixes
every rounding."""

from __future__ import annotations

import pytest
import torch

E4M3 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}


@pytest.fixture(scope="module")
def ops(pkg):
    from b200moe import experts, fp8, permute

    return type("Ops", (), {"permute": permute, "fp8": fp8, "experts": experts})


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# --------------------------------------------------------------------- SwiGLU
def swiglu_by_steps(h, limit):
    """The quantized SwiGLU in f32, one IEEE operation at a time: (E4M3 codes, scales)."""
    gate, up = h.float().chunk(2, 1)
    g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
    a = g / (1 + torch.exp(-g)) * u
    rows, width = a.shape
    b = torch.nn.functional.pad(a, (0, -width % 128)).view(rows, -1, 128)
    amax = b.abs().amax(-1).clamp_min(1e-30)
    top = torch.full_like(amax, 448.0)
    q = (b * (top / amax)[..., None]).view(rows, -1)[:, :width].to(E4M3)
    return q.view(torch.uint8), amax / top


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", [(2000, 1408), (1500, 1401), (1, 2048)])
def test_swiglu_gives_the_bits_of_its_definition(ops, dtype, rows, width):
    """f32's own exponential and division, as in the layer's SwiGLU: no code and no scale may differ."""
    h = randn(rows, rows, 2 * width, dtype=dtype) * 3
    q, scale = ops.fp8.swiglu_quantize(h)
    want_q, want_scale = swiglu_by_steps(h, 10.0)
    assert torch.equal(scale, want_scale)
    assert torch.equal(q.view(torch.uint8), want_q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", [(2000, 1408), (1500, 1401), (1, 2048)])
def test_swiglu_gradient_by_the_steps_of_its_formula(ops, dtype, rows, width):
    """d u (s (1 + g (1 - s))) and d (g s), each operation rounded to f32, the result once more: no bit may differ."""
    h, d = randn(rows, rows, 2 * width, dtype=dtype) * 4, randn(width, rows, width, dtype=dtype)
    gate, up = h.float().chunk(2, 1)
    g, u = gate.clamp(max=10.0), up.clamp(-10.0, 10.0)
    one = torch.ones((), device="cuda")
    s = one / (1 + torch.exp(-g))
    dg = torch.where(gate > 10.0, 0.0, d.float() * u * (s * (1 + g * (1 - s))))
    du = torch.where(up.abs() > 10.0, 0.0, d.float() * (g * s))
    assert torch.equal(ops.fp8.swiglu_grad(h, d), torch.cat([dg, du], 1).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [None, 3e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [128, 33])
def test_swiglu_of_the_largest_finite_gates(ops, dtype, width, limit):
    """exp(-g) is 0 there: the value is g u, finite; its gradients are d u and d g (d u is 0 past the limit)."""
    top = min(torch.finfo(dtype).max, float("inf") if limit is None else limit)
    h = torch.zeros(4, 2 * width, device="cuda", dtype=dtype)
    h[0, 5], h[1, 7], h[2, 9], h[3, 11] = torch.finfo(dtype).max, 2.5e38, 1e30, 200.0
    h[:, width:] = 0.5
    q, scale = ops.fp8.swiglu_quantize(h, limit=limit)
    got = (q.double() * scale.double().repeat_interleave(128, 1)[:, :width]).amax(1)
    gate = h[:, :width].double().clamp(max=top)
    want = (gate * 0.5).amax(1)
    assert bool(((got - want).abs() <= 4 * 2.0**-24 * want).all())  # a block's largest value is exact but for its scale
    d = torch.ones(4, width, device="cuda", dtype=dtype)
    grad = ops.fp8.swiglu_grad(h, d, limit=limit).double()
    for r, c in enumerate((5, 7, 9, 11)):
        cut = limit is not None and float(h[r, c]) > limit
        assert float(grad[r, c]) == (0.0 if cut else 0.5)
        assert abs(float(grad[r, width + c]) - float(gate[r, c])) <= 2.0**-8 * float(gate[r, c])
    assert not bool(grad.isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [256, 33])
def test_swiglu_of_low_gates(ops, dtype, width):
    """Down to -88.7 exp(-g) is finite in f32 and a large up makes the value count; below, the value is 0 (the 64-bit
    one is under 1e-36 of up)."""
    gates = [-80.0, -87.0, -87.5, -88.0, -88.25, -88.5, -89.0, -100.0, -1e4, -1e30, torch.finfo(dtype).min,
             -float("inf")]
    h = torch.zeros(len(gates), 2 * width, device="cuda", dtype=dtype)
    h[:, 3] = torch.tensor(gates, device="cuda")
    h[:, width + 3] = 1e37
    g, u = h[:, 3].double(), h[:, width + 3].double()
    s = torch.where(g < -88.7, 0.0, torch.sigmoid(g))
    g = g.clamp_min(-1e3)
    q, scale = ops.fp8.swiglu_quantize(h, limit=None)
    got = q[:, 3].double() * scale[:, 0].double()
    # the exponential's and four more roundings; below f32's normal numbers nothing is divided here
    assert bool(((got - g * s * u).abs() <= 8 * 2.0**-24 * (g * s * u).abs()).all())
    grad = ops.fp8.swiglu_grad(h, torch.ones(len(gates), width, dtype=dtype, device="cuda"), limit=None).double()
    want = u * (s + g * s * (1 - s))
    near = U[dtype] * want.abs() + 16 * 2.0**-24 * u * (s + g.abs() * s) + TINY[dtype]
    assert bool(((grad[:, 3] - want).abs() <= near).all())
    assert bool(((grad[:, width + 3] - g * s).abs() <= U[dtype] * (g * s).abs() + 2.0**-126).all())


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [10.0, None])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width", [256, 257])
def test_swiglu_of_special_values(ops, dtype, limit, width):
    """A NaN makes its block NaN and no other; an infinite value the same; a bound turns an infinity into itself."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(dtype).min
    cases = [(nan, 1.0), (1.0, nan), (inf, 1.0), (-inf, 1.0), (1.0, inf), (1.0, -inf), (low, 1.0), (low, low),
             (-inf, 0.0), (0.0, 1.0), (1.0, 0.0), (torch.finfo(dtype).tiny, torch.finfo(dtype).tiny)]
    h = torch.full((len(cases), 2 * width), 0.5, device="cuda", dtype=dtype)
    h[:, 7] = torch.tensor([c[0] for c in cases], device="cuda")
    h[:, width + 7] = torch.tensor([c[1] for c in cases], device="cuda")
    q, scale = ops.fp8.swiglu_quantize(h, limit=limit)
    v = q.double() * scale.double().repeat_interleave(128, 1)[:, :width]
    d = torch.ones(len(cases), width, device="cuda", dtype=dtype)
    grad = ops.fp8.swiglu_grad(h, d, limit=limit)
    gate, up = h.double().chunk(2, 1)
    lim = inf if limit is None else limit
    g, u = gate.clamp(max=lim).clamp_min(-1e3), up.clamp(-lim, lim)
    s = torch.sigmoid(g)
    want = g * s * u
    for r, (a, b) in enumerate(cases):
        bad = not bool(torch.isfinite(want[r, 7]))
        assert bool(v[r, :128].isnan().all()) == bad and not bool(v[r, 128:].isnan().any()), (a, b)
        if not bad:
            step = 2.0**-4 * want[r].abs() + 2.0**-10 * float(scale[r].max())
            assert bool(((v[r] - want[r]).abs() <= step * (1 + 2.0**-18) + 2.0**-20 * float(scale[r].max()) * 448).all())
        zero = torch.tensor([j not in (7, width + 7) for j in range(2 * width)], device="cuda")
        assert not bool(grad[r][zero].isnan().any()), (a, b)
    up_cut = [r for r, (_, b) in enumerate(cases) if abs(b) > lim]
    gate_cut = [r for r, (a, _) in enumerate(cases) if a > lim]
    assert not grad[up_cut, width + 7].any() and not grad[gate_cut, 7].any()
    assert grad[[0, 1], 7].isnan().all() and grad[0, width + 7].isnan() and not grad[1, width + 7].isnan()
    assert not grad[[3, 6, 8]][:, [7, width + 7]].any()  # the lowest gates: no slope


# -------------------------------------------------------------------- refusals
@pytest.mark.gpu
def test_permute_refuses_gradients_of_quantized_rows(ops):
    """A float8 tensor may require a gradient in torch; the operators have none for it.  Only the refusal is run."""
    ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    leaf = randn(0, 3, 64).to(E4M3).requires_grad_()
    cast = randn(0, 3, 64).requires_grad_().to(E4M3)
    assert leaf.requires_grad and cast.requires_grad
    for x in (leaf, cast):
        for scale in (None, torch.ones(3, 1, device="cuda")):
            with pytest.raises(ValueError, match="gradient"):
                ops.permute.permute(x, ids, 4, scale=scale)
        with torch.no_grad():
            assert torch.equal(ops.permute.permute(x, ids, 4).rows[0].float(), x[0].float())


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused(ops):
    """A dual tensor has no requires_grad: without the refusal its tangent would read as zero."""
    from torch.autograd import forward_ad

    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    w, ws = packed(0, 48, 64)
    m = ops.experts.Fp8Experts.from_weights(randn(1, 2, 64, 64), randn(2, 2, 64, 32), trainable=True)
    weights = torch.rand(4, 2, device="cuda")
    row, _ = ops.permute.sort_routes(ids, 2)
    with forward_ad.dual_level():
        dual = lambda v: forward_ad.make_dual(v, torch.ones_like(v))  # noqa: E731
        x, rows, half = dual(randn(3, 4, 64)), dual(randn(4, 8, 64)), dual(randn(5, 4, 64, dtype=torch.bfloat16))
        calls = [lambda: ops.permute.permute(x, ids, 2), lambda: ops.permute.unpermute(rows, row),
                 lambda: ops.permute.unpermute(randn(4, 8, 64), row, dual(weights)),
                 lambda: ops.fp8.linear(x, w, ws), lambda: ops.fp8.quantize(x), lambda: ops.fp8.swiglu_quantize(x),
                 lambda: ops.fp8.swiglu_grad(x, randn(6, 4, 32)), lambda: m(half, ids, weights),
                 lambda: m(randn(7, 4, 64, dtype=torch.bfloat16), ids, dual(weights))]
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
        y = randn(8, 4, 64).requires_grad_()  # a tangent of the incoming gradient
        for out in (ops.permute.permute(y, ids, 2).rows, ops.fp8.linear(y, w, ws),
                    ops.permute.unpermute(y, torch.tensor([[0], [1], [2], [3]], dtype=torch.int32, device="cuda"))):
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, y, dual(torch.ones_like(out.detach())))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 2**32 + 5, 1), (1, 2**31, 1), (2**16, 1, 1), (2**23, 1)])
def test_weights_past_the_kernels_sizes_are_refused(ops, shape):
    """Every axis counts, the middle one of three too: 2^32 + 5 cut to 32 bits would be five rows."""
    w = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="too large"):
        ops.fp8.quantize_weight(w)
    del w
    q = torch.empty(shape, dtype=torch.uint8, device="cuda").view(E4M3)
    scale = torch.empty(*shape[:-2], -(-shape[-2] // 128), 1, device="cuda")
    with pytest.raises(ValueError, match="too large"):
        ops.fp8.transpose_weight(q, scale)


# -------------------------------------------------------------------- products
def packed(seed, *shape):
    """E4M3 values of any size with a scale per 128 x 128 block."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q = (60 * torch.randn(*shape, generator=g, device="cuda")).clamp(-448, 448).to(E4M3)
    n, k = -(-shape[-2] // 128), -(-shape[-1] // 128)
    return q, torch.rand(*shape[:-2], n, k, generator=g, device="cuda") * 1e-3 + 1e-4


def check_product(got, q, scale, w, w_scale):
    """Against 64 bits: 128 products a block, the scales' two roundings and one addition per block, each losing at
    most 2^-23 of the sum of magnitudes, and the output's own rounding."""
    k, n = q.shape[1], w.shape[0]
    a = q.double() * scale.double().repeat_interleave(128, 1)[:, :k]
    b = w.double() * w_scale.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want, mag = a @ b.T, a.abs() @ b.abs().T
    bound = (128 + -(-k // 128) + 4) * 2.0**-23 * mag + U[got.dtype] * want.abs() + TINY[got.dtype]
    assert got.shape == want.shape
    excess = (got.double() - want).abs() - bound
    assert bool((excess <= 0).all()), f"worst excess {float(excess.max()):.3e}"


@pytest.mark.gpu
def test_long_product_gives_the_same_bits_every_time(ops):
    """Tiles of 256 columns hand their two TMEM buffers over 64 times a tile: a sum that met the next block's values
    would differ from call to call."""
    q, scale = ops.fp8.quantize(randn(1, 2560, 8192))
    w, ws = packed(2, 2304, 8192)
    first = ops.fp8.matmul(q, scale, w, ws, out_dtype=torch.float32)
    check_product(first, q, scale, w, ws)
    for _ in range(20):
        assert torch.equal(ops.fp8.matmul(q, scale, w, ws, out_dtype=torch.float32), first)
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,head,tail", [([3, 0, 5], 4, 0), ([0, 0], 7, 3), ([200, 150], 130, 20),
                                              ([3000, 0, 2500], 700, 11)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_rows_before_the_first_expert_are_zeros(ops, counts, head, tail, out_dtype):
    """A part of the experts' offsets: the rows of the experts before it have none here."""
    n, k, rows = 1064, 144, head + sum(counts) + tail
    off = torch.tensor([head, *counts], device="cuda").cumsum(0).to(torch.int32)
    q, scale = ops.fp8.quantize(randn(rows, rows, k))
    w, ws = packed(head, len(counts), n, k)
    for r in (slice(0, head), slice(rows - tail, rows)):
        q.view(torch.uint8)[r] = 0x7F
    torch.full((rows, n), float("nan"), dtype=out_dtype, device="cuda")  # what the output's memory held before
    got = ops.fp8.grouped_matmul(q, scale, off, w, ws, out_dtype=out_dtype)
    assert not got[:head].any() and not got[rows - tail:].any()
    for e in range(len(counts)):
        r = slice(int(off[e]), int(off[e + 1]))
        if counts[e]:
            check_product(got[r], q[r], scale[r], w[e], ws[e])
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2500, 2049, 144), (2500, 2100, 256), (4801, 1000, 400), (2500, 2056, 2064)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_wide_tiles_that_end_inside(ops, m, n, k, out_dtype):
    """Tiles of 128 x 256 (148 of them at least) whose last columns, rows and K block are partial: whole pieces leave by
    clipped copies, odd rows by elements."""
    q, scale = ops.fp8.quantize(randn(m + n, m, k))
    w, ws = packed(k, n, k)
    check_product(ops.fp8.matmul(q, scale, w, ws, out_dtype=out_dtype), q, scale, w, ws)
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1023, 1064, 1280])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_wide_tiles_by_expert(ops, n, out_dtype):
    """Experts that begin and end inside a tile's 32-row copies, every row looked at."""
    counts, k, tail = [700, 1, 0, 129, 333, 2000, 31, 64, 95, 500, 32, 128], 272, 19
    off = torch.tensor([0, *counts], device="cuda").cumsum(0).to(torch.int32)
    rows = sum(counts) + tail
    q, scale = ops.fp8.quantize(randn(n, rows, k))
    w, ws = packed(n, len(counts), n, k)
    got = ops.fp8.grouped_matmul(q, scale, off, w, ws, out_dtype=out_dtype)
    for e, c in enumerate(counts):
        r = slice(int(off[e]), int(off[e + 1]))
        if c:
            check_product(got[r], q[r], scale[r], w[e], ws[e])
    assert not got[rows - tail:].any()
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 20, 33])
@pytest.mark.parametrize("k", [12544, 12560, 16384, 16400, 32768, 32784])
def test_longest_k_of_each_kernel(ops, m, k):
    """One matrix: eight rows' values fill shared memory up to K 12544, the scales of 32 rows up to 16384, of 16 up to
    32768; past each the next kernel takes over."""
    q, scale = ops.fp8.quantize(randn(m, m, k))
    w, ws = packed(k, 200, k)
    check_product(ops.fp8.matmul(q, scale, w, ws), q, scale, w, ws)
    x = randn(k, m, k, dtype=torch.bfloat16)
    q, scale = ops.fp8.quantize(x)
    check_product(ops.fp8.linear(x, w, ws), q, scale, w, ws)
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("k", [16384, 16400])
def test_longest_k_by_expert(ops, k):
    counts = [5, 0, 20, 33]
    off = torch.tensor([0, *counts], device="cuda").cumsum(0).to(torch.int32)
    q, scale = ops.fp8.quantize(randn(k, sum(counts), k))
    w, ws = packed(k, len(counts), 300, k)
    got = ops.fp8.grouped_matmul(q, scale, off, w, ws)
    for e, c in enumerate(counts):
        r = slice(int(off[e]), int(off[e + 1]))
        if c:
            check_product(got[r], q[r], scale[r], w[e], ws[e])
    ops.fp8.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8])
@pytest.mark.parametrize("n,k", [(4736, 2064), (4737, 2064), (9472, 272), (9473, 272), (2368, 6400), (2369, 6400)])
def test_few_rows_at_the_end_of_a_wave(ops, m, n, k):
    """The few-row kernel's last item that has a CTA of its own, and the first that has none."""
    w, ws = packed(n, n, k)
    x = randn(k, m, k, dtype=torch.bfloat16)
    q, scale = ops.fp8.quantize(x)
    check_product(ops.fp8.matmul(q, scale, w, ws, out_dtype=torch.float32), q, scale, w, ws)
    check_product(ops.fp8.linear(x, w, ws), q, scale, w, ws)
    ops.fp8.check_errors()


# ---------------------------------------------------------------------- errors
@pytest.mark.gpu
def test_no_error_is_lost_between_streams(ops):
    """An error that one stream's kernel reports while another stream reads the word is seen by that read or the next."""
    from b200moe._lib import B200MoeError

    rows, bad = torch.ones(2, 8, device="cuda"), torch.tensor([[0, 99]], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def reported():
        try:
            ops.permute.check_errors()
        except B200MoeError:
            return 1
        return 0

    for i in range(2000):
        with torch.cuda.stream(side):
            torch.cuda._sleep(500 * (i % 100))  # up to some 25 us, past the read below
            ops.permute.unpermute(rows, bad)
        seen = reported()
        side.synchronize()
        assert seen + reported() == 1, i
    assert reported() == 0


# --------------------------------------------------------------------- experts
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_router_weights_learn_without_transposed_weights(ops, dtype):
    """Their gradient is <grad, y>: the same bits with and without the weights that only the tokens' gradient reads."""
    t, k, e, h, i = 21, 3, 6, 128, 96
    w13, w2 = 0.05 * randn(1, e, 2 * i, h), 0.05 * randn(2, e, h, i)
    x, ids = randn(3, t, h, dtype=dtype), torch.randint(-1, e, (t, k), dtype=torch.int32, device="cuda")
    grad, got = randn(4, t, h, dtype=dtype), []
    for trainable in (False, True):
        m = ops.experts.Fp8Experts.from_weights(w13, w2, trainable=trainable)
        w = torch.rand(t, k, generator=torch.Generator("cuda").manual_seed(5), device="cuda").requires_grad_()
        got += torch.autograd.grad(m(x, ids, w), w, grad)
        if not trainable:
            with pytest.raises(ValueError, match="trainable"):
                m(x.clone().requires_grad_(), ids, w)
    assert torch.equal(*got) and bool(got[0].any()) and not got[0][ids < 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,e,h,i", [(1, 4, 16, 512, 256), (70, 6, 16, 512, 352), (900, 4, 8, 256, 128)])
def test_fp8_experts_in_f16(ops, t, k, e, h, i):
    """The whole path in f16, in the norm within 2^-8: f16's roundings take 2^-11 each, and the share of values whose
    32-bit form falls on the other side of an E4M3 boundary (2^-20 / 2^-4 of them, 2^-3 off) less than that."""
    from test_gpu_fp8_experts import dequantize, plain_experts, rng, routes

    m = ops.experts.Fp8Experts.from_weights(0.05 * randn(1, e, 2 * i, h), 0.05 * randn(2, e, h, i), trainable=True)
    x, ids = randn(3, t, h, dtype=torch.float16), routes(rng(t), t, k, e, 0.1)
    w, grad = torch.rand(t, k, generator=rng(t + 1), device="cuda"), randn(4, t, h, dtype=torch.float16)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = m(xr, ids, wr)
    gx, gw = torch.autograd.grad(out, (xr, wr), grad)
    assert out.dtype == gx.dtype == torch.float16 and torch.equal(out, m(x, ids, w))
    wide = lambda q, s: dequantize(q, s.repeat_interleave(128, -2)[..., : q.shape[-2], :])  # noqa: E731
    want = plain_experts(x, ids, w, wide(m.w13, m.w13_scale), wide(m.w2, m.w2_scale), 10.0, grad)
    for got, ref in zip((out, gx, gw), want):
        assert float((got.detach().double() - ref).norm()) <= 2.0**-8 * float(ref.norm())
    ops.fp8.check_errors()
