"""The norm (``norm``) where ``test_gpu_norm`` does not reach: widths of two and four pieces per thread and their gradients,
E4M3 codes against 64 bits, calls on two streams, a captured backward pass.  Tolerances are that file's."""

from __future__ import annotations

import pytest
import torch
from test_gpu_norm import DTYPES, inputs, ops, randn  # noqa: F401
from test_gpu_norm import test_gradients as check_gradients
from test_gpu_norm import test_norm as check_norm
from test_gpu_norm import test_quantized_rows_are_those_of_the_norm as check_quantized


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("res,weight_f32", [("none", True), ("same", False), ("f32", True)])
@pytest.mark.parametrize("m,h", [(5, 4097), (3, 4104), (300, 5120), (40, 6144), (9, 7168), (2, 8191), (400, 8192), (2, 8200),
                                 (3, 16376), (150, 16384)])
def test_widths_of_several_pieces(ops, dtype, res, weight_f32, m, h):  # noqa: F811
    check_norm(ops, dtype, res, weight_f32, m, h)
    check_gradients(ops, dtype, res, weight_f32, m, h)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp8", "nvfp4", "mxfp4"])
@pytest.mark.parametrize("res", ["none", "f32"])
@pytest.mark.parametrize("m,h", [(3, 4128), (300, 5120), (9, 7168), (2, 12288)])
def test_quantized_widths_of_several_pieces(ops, fmt, res, m, h):  # noqa: F811
    for dtype in DTYPES:
        check_quantized(ops, fmt, dtype, res, m, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h", [(64, 4096), (40, 1401), (7, 4097), (5, 8191), (300, 96)])
def test_e4m3_codes_against_64_bits(ops, dtype, m, h):  # noqa: F811
    """A scale is off by less than 2^-18; a code is a nearest one of the 64-bit quotient up to 2^-17 of it (y's 2^-19, the
    block's maximum's and five roundings).  Exact ties, in which the root cancels, may fall either way."""
    x, r, w = inputs(m, h, dtype, "same", False)
    (q, scale), total, _ = ops.norm.rms_norm_quantize(x, w, r)
    s = total.double()
    y = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
    b = torch.cat([y, y.new_zeros(m, -h % 128)], 1).view(m, -1, 128)
    want = b.abs().amax(2).clamp_min(1e-30) / 448
    assert bool(((scale.double() - want).abs() <= 2.0**-18 * want).all())
    t = (b / want[..., None]).view(m, -1)[:, :h].abs()
    half = torch.ldexp(torch.ones_like(t), torch.frexp(t)[1].clamp_min(-5) - 5)
    off = (q.double().abs() - t).abs()
    assert bool((off <= half + 2.0**-17 * t).all())
    assert bool(((q.double() == 0) | (torch.signbit(q.double()) == torch.signbit(y))).all())


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(ops):  # noqa: F811
    """Alternating calls with inputs of their own: the weight's gradient passes through a workspace."""
    sets = [(inputs(700 + i, 2048, torch.bfloat16, "same", True), randn(i, 700 + i, 2048, dtype=torch.bfloat16)) for i in range(4)]

    def run(i):
        (x, r, w), dy = sets[i]
        n = ops.norm.rms_norm_quantize(x, w, r, format="nvfp4", keep=True)
        return (n.sum, n.y, n.rows.record, *ops.norm.rms_norm_grad(n.sum, dy, w, dy))

    want = [run(i) for i in range(4)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for j in range(40):
        with torch.cuda.stream(streams[j % 2]):
            got.append((j % 4, run(j % 4)))
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


@pytest.mark.gpu
def test_captured_training_step(ops):  # noqa: F811
    """Forward and backward of the autograd function in a graph, replayed on other inputs."""
    x, r, w = (t.requires_grad_() for t in inputs(130, 1024, torch.bfloat16, "same", True))
    dy, ds = randn(5, 130, 1024, dtype=torch.bfloat16), randn(6, 130, 1024, dtype=torch.bfloat16)

    def step():
        y, total = ops.norm.rms_norm(x, w, r)
        return (y, total, *torch.autograd.grad((y, total), (x, r, w), (dy, ds)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    with torch.no_grad():
        x.copy_(randn(7, 130, 1024))
        dy.copy_(randn(8, 130, 1024))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
