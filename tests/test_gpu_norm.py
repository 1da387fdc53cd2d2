"""Residual RMS norm on the GPU against the formulas in 64 bits (csrc/norm.cu).

Tolerances, fixed before the first run.  y: one BF16 rounding, 2^-8 of the value, and fewer than 2^7 FP32 roundings
of 2^-24 on the way (the longest chain adds 32 squares per thread and then 5 + 16 partial sums).  dx: the same against
the size of its three summands.  dgamma: one BF16 rounding and an FP32 sum of `rows` products whose error is at most
(rows + 64) 2^-24 of the sum of their sizes.  The stream h and the MXFP8 bytes are exact."""
import numpy as np
import pytest
import torch

from fuse_b200 import _native as N
from fuse_b200 import api, block

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
EPS = 1e-6


def make(rows, hidden, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x, res = ((scale * torch.randn(rows, hidden, generator=gen, device=DEV)).to(BF16) for _ in range(2))
    gamma = (1.0 + 0.3 * torch.randn(hidden, generator=gen, device=DEV)).to(BF16)
    dy, dh = (torch.randn(rows, hidden, generator=gen, device=DEV).to(BF16) for _ in range(2))
    return x, res, gamma, dy, dh


def forward64(h, gamma, eps=EPS):
    h, g = h.double(), gamma.double()
    return h * torch.rsqrt(h.square().mean(1, keepdim=True) + eps) * g


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()))


def check_y(y, want):
    within(y, want, want.abs() * (2.0 ** -8 + 2.0 ** -17) + 2.0 ** -134, "y")


SHAPES = [(1, 8), (3, 32), (5, 256), (7, 264), (4, 520), (130, 1024), (9, 1032), (300, 4096), (33, 5120), (2, 8192),
          (5, 8200), (4, 16384), (0, 64), (700, 40)]


@pytest.mark.parametrize("rows,hidden", SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_forward(rows, hidden, with_residual):
    x, res, gamma, _, _ = make(rows, hidden, rows + hidden)
    y, h = block.rms_norm(x, gamma, res if with_residual else None)
    want_h = (x.float() + res.float()).to(BF16) if with_residual else x
    assert torch.equal(h, want_h) and (with_residual or h is x)
    check_y(y, forward64(want_h, gamma))


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e18])
def test_forward_at_the_ends_of_the_range(scale):
    x, res, gamma, _, _ = make(6, 512, 3, scale)
    y, h = block.rms_norm(x, gamma, res)
    check_y(y, forward64(h, gamma))
    assert torch.isfinite(y).all()


def test_rows_do_not_reach_one_another():
    x, res, gamma, _, _ = make(260, 640, 4)
    want, _ = block.rms_norm(x, gamma, res)
    x = x.clone()
    x[7], x[100, 3] = float("nan"), float("inf")
    y, _ = block.rms_norm(x, gamma, res)
    keep = torch.ones(260, dtype=torch.bool, device=DEV)
    keep[[7, 100]] = False
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[7]).all()


@pytest.mark.parametrize("rows,hidden", [(1, 32), (5, 160), (128, 256), (130, 1024), (257, 4096), (3, 5120), (131, 8224), (2, 16384)])
def test_mxfp8_bytes_are_those_of_the_bf16_output(rows, hidden):
    x, res, gamma, _, _ = make(rows, hidden, 5)
    gamma[::7] = 0.0
    x[0], res[0] = 0.0, 0.0
    y, h, data, scales = block.rms_norm(x, gamma, res, mxfp8=True)
    check_y(y, forward64(h, gamma))
    want_data = torch.empty_like(data)
    want_scales = torch.full_like(scales, 127)
    assert api.quantize_mxfp8(y.data_ptr(), hidden, rows, hidden, want_data.data_ptr(), want_scales.data_ptr()) == 0
    torch.cuda.synchronize()
    assert torch.equal(data, want_data) and torch.equal(scales, want_scales)
    h2, data2, scales2 = block.rms_norm_mxfp8(x, gamma, res)
    assert torch.equal(h2, h) and torch.equal(data2, data) and torch.equal(scales2, scales)


@pytest.mark.parametrize("rows,hidden", [s for s in SHAPES if s[0]] + [(1500, 2048)])
@pytest.mark.parametrize("with_stream", [True, False])
def test_backward(rows, hidden, with_stream):
    x, res, gamma, dy, dh = make(rows, hidden, rows * 3 + hidden)
    x, res, gamma = (t.requires_grad_() for t in (x, res, gamma))
    y, h = block.rms_norm(x, gamma, res)
    if with_stream:
        dx, dres, dgamma = torch.autograd.grad((y, h), (x, res, gamma), (dy, dh))
    else:
        dx, dres, dgamma = torch.autograd.grad(y, (x, res, gamma), dy)
    assert torch.equal(dx, dres)
    hh, g, d = h.detach().double(), gamma.detach().double(), dy.double()
    r = torch.rsqrt(hh.square().mean(1, keepdim=True) + EPS)
    n, dn = hh * r, d * g
    mean = (dn * n).mean(1, keepdim=True)
    past = dh.double() if with_stream else torch.zeros_like(d)
    want = past + r * (dn - n * mean)
    size = past.abs() + r * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True))
    within(dx, want, want.abs() * 2.0 ** -8 + size * 2.0 ** -16 + 2.0 ** -134, "dx")
    want = (d * n).sum(0)
    within(dgamma, want, want.abs() * 2.0 ** -8 + (d * n).abs().sum(0) * (rows + 192) * 2.0 ** -24, "dgamma")


def test_backward_against_differences():
    x, res, gamma, dy, dh = make(6, 320, 11)
    leaves = [t.clone().requires_grad_() for t in (x, gamma)]
    y, _ = block.rms_norm(leaves[0], leaves[1])
    grads = torch.autograd.grad(y, leaves, dy)
    gen = torch.Generator(device=DEV).manual_seed(12)
    for which, grad in enumerate(grads):
        base = [x.double(), gamma.double()]
        step = torch.randn(base[which].shape, generator=gen, device=DEV, dtype=torch.float64)
        def at(e):
            moved = list(base)
            moved[which] = moved[which] + e * step
            return (forward64(moved[0], moved[1]) * dy.double()).sum()
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        tol = (grad.double().abs() * step.abs()).sum() * 2.0 ** -8 + 1e-6 * slope.abs() + 1e-6
        assert (slope - (grad.double() * step).sum()).abs() <= tol


def test_backward_takes_gradients_as_autograd_makes_them():
    x, _, gamma, _, _ = make(40, 264, 13)
    x, gamma = x.requires_grad_(), gamma.requires_grad_()
    y, _ = block.rms_norm(x, gamma)
    y.sum().backward()  # an expanded gradient, row stride 0
    dx, dgamma = x.grad.clone(), gamma.grad.clone()
    y, _ = block.rms_norm(x, gamma)
    ones = torch.ones_like(y)
    want = torch.autograd.grad(y, (x, gamma), ones)
    assert torch.equal(dx, want[0]) and torch.equal(dgamma, want[1])
    y, h = block.rms_norm(x, gamma, x.detach())
    dx, = torch.autograd.grad(h, x, ones)  # past the norm alone
    assert torch.equal(dx, ones)


def test_backward_is_the_same_every_time():
    x, res, gamma, dy, dh = make(3001, 1536, 14)
    x, gamma = x.requires_grad_(), gamma.requires_grad_()
    first = None
    for _ in range(3):
        y, h = block.rms_norm(x, gamma, res)
        grads = torch.autograd.grad((y, h), (x, gamma), (dy, dh))
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(first, grads))


def test_strided_rows_and_in_place_outputs():
    wide = torch.randn(50, 1024, device=DEV).to(BF16)
    x, res = wide[:, 64:576], wide[:, 512:1024].clone()
    gamma = torch.randn(512, device=DEV).to(BF16)
    y, h = block.rms_norm(x, gamma, res)
    want_y, want_h = block.rms_norm(x.contiguous(), gamma, res)
    assert torch.equal(y, want_y) and torch.equal(h, want_h)
    # the C entry: the stream written over the residual, y over the input, neighbours untouched
    before = wide.clone()
    p = N.RmsNormParams(input=x.data_ptr(), residual=res.data_ptr(), gamma=gamma.data_ptr(), residual_output=res.data_ptr(),
                        output=x.data_ptr(), input_stride=1024, residual_stride=-1, residual_output_stride=-1,
                        output_stride=1024, rows=50, hidden=512, epsilon=EPS)
    assert api.launch_rms_norm(p) == 0
    torch.cuda.synchronize()
    assert torch.equal(x, want_y) and torch.equal(res, want_h)
    assert torch.equal(wide[:, :64], before[:, :64]) and torch.equal(wide[:, 576:], before[:, 576:])


def test_refusals():
    x, res, gamma, _, _ = make(4, 256, 15)
    for call in (lambda: block.rms_norm(x, gamma[:128]), lambda: block.rms_norm(x, gamma.float()),
                 lambda: block.rms_norm(x, gamma, res[:3]), lambda: block.rms_norm(x.t(), gamma),
                 lambda: block.rms_norm(x[:, :40], gamma[:40], mxfp8=True)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        block.rms_norm(x.view(-1)[4:1004].view(5, 200), gamma[:200])  # not on a 16-byte boundary
    with pytest.raises(RuntimeError):
        block.rms_norm_mxfp8(x.clone().requires_grad_(), gamma)
    p = N.RmsNormBackwardParams(grad_output=x.data_ptr(), stream_input=x.data_ptr(), gamma=gamma.data_ptr(),
                                grad_input=res.data_ptr(), grad_gamma=gamma.data_ptr(), grad_output_stride=-1,
                                stream_input_stride=-1, grad_stream_stride=-1, grad_input_stride=-1, rows=4, hidden=256,
                                epsilon=EPS)
    assert api.launch_rms_norm_backward(p) == N.CUDA_ERROR_INVALID_VALUE  # no workspace
    torch.cuda.synchronize()


def test_captured_and_on_another_stream():
    x, res, gamma, dy, dh = make(200, 2048, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, h = block.rms_norm(x, gamma, res)
    torch.cuda.current_stream().wait_stream(side)
    want, _ = block.rms_norm(x, gamma, res)
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    xs = x.clone().requires_grad_()
    with torch.cuda.graph(graph):
        y, h = block.rms_norm(xs, gamma, res)
        dx, = torch.autograd.grad((y, h), xs, (dy, dh))
    with torch.no_grad():
        xs.copy_(res)
    graph.replay()
    torch.cuda.synchronize()
    fresh = res.clone().requires_grad_()
    want_y, want_h = block.rms_norm(fresh, gamma, res)
    want_dx, = torch.autograd.grad((want_y, want_h), fresh, (dy, dh))
    assert torch.equal(y, want_y) and torch.equal(dx, want_dx)


def test_backward_of_no_rows():
    x, gamma = torch.empty(0, 512, dtype=BF16, device=DEV, requires_grad=True), torch.ones(512, dtype=BF16, device=DEV, requires_grad=True)
    y, h = block.rms_norm(x, gamma)
    dx, dgamma = torch.autograd.grad(y, (x, gamma), torch.empty_like(y))
    assert dx.shape == (0, 512) and (dgamma == 0).all()


def test_gradients_past_the_range_of_fp32_squares():
    x, _, gamma, dy, _ = make(5, 640, 17, 1e25)
    x = x.requires_grad_()
    y, _ = block.rms_norm(x, gamma)
    dx, = torch.autograd.grad(y, x, dy)
    h, d = x.detach().double(), dy.double() * gamma.double()
    r = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    n = h * r
    want = r * (d - n * (d * n).mean(1, keepdim=True))
    size = r * (d.abs() + n.abs() * (d * n).abs().mean(1, keepdim=True))
    within(dx, want, want.abs() * 2.0 ** -8 + size * 2.0 ** -16 + 2.0 ** -134, "dx")
