"""Rotary positions on the GPU against the formulas in 64 bits (csrc/rotary.cu).

Tolerance, fixed before the first run: one BF16 rounding, 2^-8 of the value; the angle is a 32-bit fraction of a half
turn put in FP32 (pi 2^-25) and sincospif, the products and the sum add a few roundings of 2^-24: 2^-20 of m (|a| + |b|)."""
import math

import pytest
import torch

from fuse_b200 import block

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def expected(x, spec, head_dim, positions, sign=1.0):
    """(value, m (|a| + |b|)) in 64 bits."""
    f, m = spec.frequencies()
    angle = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=DEV)
    c, s = (torch.cos(angle) * m)[:, None], (torch.sin(angle) * m * sign)[:, None]
    x = x.double().view(x.shape[0], x.shape[1] // head_dim, head_dim)
    out, size = x.clone(), x.abs()
    rd = spec.rotary_dim
    first, second = (slice(0, rd, 2), slice(1, rd, 2)) if spec.interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = m * (a.abs() + b.abs())
    return out.flatten(1), size.flatten(1)


def check(got, x, spec, head_dim, positions, sign=1.0):
    want, size = expected(x, spec, head_dim, positions, sign)
    bad = ~((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -20)
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()))


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(BF16)


SPECS = {
    "none": dict(), "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=4.0),
    "wavelength": dict(scaling="wavelength", factor=8.0, original_context=8192),
    "yarn": dict(scaling="yarn", factor=16.0, original_context=4096),
}
# rows, q_heads, kv_heads, head_dim, rotary_dim
SHAPES = [(1, 4, 1, 128, 128), (7, 3, 1, 64, 64), (257, 8, 2, 128, 64), (33, 5, 5, 256, 256), (50, 2, 2, 96, 48),
          (19, 3, 1, 80, 40), (40, 4, 2, 20, 6), (5, 64, 8, 128, 32), (3, 200, 0, 128, 128), (11, 0, 4, 64, 16), (0, 2, 1, 64, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", list(SPECS))
def test_forward(shape, interleaved, scaling):
    rows, hq, hk, d, rd = shape
    spec = block.Rotary(rd, 10000.0, interleaved, **SPECS[scaling])
    q, k = randn(rows, hq * d, seed=1) if hq else None, randn(rows, hk * d, seed=2) if hk else None
    seq, start = max(1, rows // 2), 12345
    qo, ko = block.rotary(q, k, spec, head_dim=d, seq_len=seq, start=start)
    positions = start + torch.arange(rows, device=DEV) % seq
    for got, x in ((qo, q), (ko, k)):
        if x is None:
            assert got is None
        else:
            check(got, x, spec, d, positions)
            kept = x.view(rows, x.shape[1] // d, d)[..., rd:]
            assert torch.equal(got.view(rows, x.shape[1] // d, d)[..., rd:], kept)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", [(64, 4, 1, 128, 128), (9, 2, 1, 24, 24)])
def test_given_and_far_positions(dtype, shape):
    rows, hq, hk, d, rd = shape
    spec = block.Rotary(rd, 500000.0)
    q, k = randn(rows, hq * d, seed=3), randn(rows, hk * d, seed=4)
    # near, far (a million and more, up to the end of 31 bits), negative, repeated
    positions = torch.randint(0, 1 << 20, (rows,), device=DEV)
    positions[:6] = torch.tensor([0, 1, (1 << 31) - 1, 1 << 30, -5, 1048576], device=DEV)
    positions = positions.to(dtype)
    qo, ko = block.rotary(q, k, spec, head_dim=d, positions=positions)
    # 64-bit cosines of an angle of 2^31 radians are themselves off by 2^31 2^-53 = 2^-22 of a radian
    want, size = expected(q, spec, d, positions)
    assert ((qo.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -19).all()
    want, size = expected(k, spec, d, positions)
    assert ((ko.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -19).all()


def test_start_past_32_bits_turns_by_whole_numbers():
    spec = block.Rotary(64)
    q = randn(20, 128, seed=5)
    a, _ = block.rotary(q, None, spec, head_dim=64, start=(1 << 33) + 7)
    b, _ = block.rotary(q, None, spec, head_dim=64, positions=torch.arange(20, device=DEV) + (1 << 33) + 7)
    assert torch.equal(a, b)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(128, 128), (128, 32), (40, 24)])
def test_gradient_is_the_adjoint(interleaved, d, rd):
    rows = 37
    spec = block.Rotary(rd, 10000.0, interleaved, **SPECS["yarn"])
    q, k = randn(rows, 4 * d, seed=6).requires_grad_(), randn(rows, 2 * d, seed=7).requires_grad_()
    dq, dk = randn(rows, 4 * d, seed=8), randn(rows, 2 * d, seed=9)
    positions = torch.arange(rows, device=DEV) * 1000
    qo, ko = block.rotary(q, k, spec, head_dim=d, positions=positions)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    check(gq, dq, spec, d, positions, -1.0)
    check(gk, dk, spec, d, positions, -1.0)
    # against differences of the 64-bit forward along a direction (the map is linear: any step does)
    step = torch.randn(rows, 4 * d, device=DEV, dtype=torch.float64)
    slope = (expected(step, spec, d, positions)[0] * dq.double()).sum()
    tol = (gq.double().abs() * step.abs()).sum() * 2.0 ** -8 + 1e-3
    assert (slope - (gq.double() * step).sum()).abs() <= tol
    qo, ko = block.rotary(q, k, spec, head_dim=d, positions=positions)
    only, = torch.autograd.grad(qo, q, torch.ones_like(qo[:1, :1]).expand_as(qo))  # one output, an expanded gradient
    check(only, torch.ones_like(qo), spec, d, positions, -1.0)


def test_in_place_strided_and_unaligned():
    d, spec = 64, block.Rotary(64, interleaved=True)
    wide = randn(30, 10 * d, seed=10)
    q, k = wide[:, :4 * d], wide[:, 6 * d:8 * d]
    want = block.rotary(q, k, spec, head_dim=d, start=3)
    keep = wide.clone()
    block.rotary_(q, k, spec, head_dim=d, start=3)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(wide[:, 4 * d:6 * d], keep[:, 4 * d:6 * d]) and torch.equal(wide[:, 8 * d:], keep[:, 8 * d:])
    odd = torch.zeros(30 * (4 * d + 1) + 1, dtype=BF16, device=DEV)[1:].view(30, 4 * d + 1)[:, :4 * d]
    odd.copy_(keep[:, :4 * d])
    block.rotary_(odd, None, spec, head_dim=d, start=3)
    assert torch.equal(odd, want[0])
    with pytest.raises(RuntimeError):
        block.rotary_(q.clone().requires_grad_(), None, spec, head_dim=d)


def test_turning_back_and_zero():
    spec = block.Rotary(128)
    q = randn(64, 512, seed=11)
    same, _ = block.rotary(q, None, spec, head_dim=128, seq_len=1)  # position 0 everywhere
    assert torch.equal(same, q)


def test_refusals():
    q = randn(8, 256, seed=12)
    for call in (lambda: block.rotary(q, None, block.Rotary(64), head_dim=100),
                 lambda: block.rotary(q, q[:4], block.Rotary(64), head_dim=64),
                 lambda: block.rotary(q, None, block.Rotary(64), head_dim=64, positions=torch.zeros(7, device=DEV, dtype=torch.int64)),
                 lambda: block.rotary(q, None, block.Rotary(64), head_dim=64, positions=torch.zeros(8, device=DEV)),
                 lambda: block.rotary(q.float(), None, block.Rotary(64), head_dim=64)):
        with pytest.raises(ValueError):
            call()
    for spec in (block.Rotary(128), block.Rotary(63), block.Rotary(64, scaling="yarn", factor=4.0)):
        with pytest.raises(RuntimeError):
            block.rotary(q, None, spec, head_dim=64)


def test_captured():
    spec = block.Rotary(128)
    q, positions = randn(100, 512, seed=13), torch.arange(100, device=DEV)
    graph = torch.cuda.CUDAGraph()
    block.rotary(q, None, spec, head_dim=128, positions=positions)
    with torch.cuda.graph(graph):
        out, _ = block.rotary(q, None, spec, head_dim=128, positions=positions)
    positions.add_(777)
    graph.replay()
    torch.cuda.synchronize()
    check(out, q, spec, 128, positions)
