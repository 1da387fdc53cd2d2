"""Rotary positions past 32 bits against whole-number arithmetic on the host (csrc/rotary.cu takes p f_i / 2 pi modulo 1 as one
64-bit product).

The FP64 frequency that Rotary.frequencies() gives is a rational number; p f_i / 2 pi modulo 1 is taken of it with 60 digits of pi.
Tolerance, fixed before the first run: one BF16 rounding, 2^-8 of the value.  The 64-bit fraction of a turn per position is
cut off at 2^-64 and comes from a quotient of 64 bits, together below 2^-63: 2 pi |p| 2^-63 of a radian.  The product's high word is cut
off at 2^-32 of a turn and rounded to FP32 (pi 2^-24 at most); the hardware's sine and cosine are within 2^-21.1 (absolute)
in [-pi, pi]; products and sum add a few roundings of 2^-24: 2^-19 of m (|a| + |b|) together."""
import math
from fractions import Fraction

import pytest
import torch

from fuse_b200 import block

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(BF16)


def check(got, x, spec, d, positions):
    f, m = spec.frequencies()
    angles = [[2 * math.pi * float(p * Fraction(v) / TWO_PI % 1) for v in f] for p in positions]
    angle = torch.tensor(angles, dtype=torch.float64, device=DEV)
    c, s = (torch.cos(angle) * m)[:, None], (torch.sin(angle) * m)[:, None]
    far = 2 * math.pi * 2.0 ** -63 * torch.tensor([float(abs(p)) for p in positions], dtype=torch.float64, device=DEV)[:, None, None]
    half = spec.rotary_dim // 2
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if spec.interleaved else (slice(0, half), slice(half, 2 * half))
    x, got = (t.double().view(len(positions), -1, d) for t in (x, got))
    a, b = x[..., first], x[..., second]
    size = m * (a.abs() + b.abs()) * (2.0 ** -19 + far)
    for want, part in ((a * c - b * s, first), (a * s + b * c, second)):
        error = (got[..., part] - want).abs()
        assert (error <= want.abs() * 2.0 ** -8 + size).all(), float((error - want.abs() * 2.0 ** -8).max())


FAR = [(1 << 32) - 1, 1 << 32, (1 << 32) + 1, (1 << 33) + 7, -1, -(1 << 31) - 5, -(1 << 32) - 3, (1 << 40) + 12345, -(1 << 41) - 77, (1 << 44) + 1, 0]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(128, 128), (24, 24)])  # in vectors, and pair by pair
@pytest.mark.parametrize("kw", [dict(), dict(scaling="wavelength", factor=8.0, original_context=8192), dict(scaling="yarn", factor=16.0, original_context=4096)])
def test_given_positions(interleaved, d, rd, kw):
    spec = block.Rotary(rd, 500000.0, interleaved, **kw)
    q, k = randn(len(FAR), 3 * d, seed=1), randn(len(FAR), d, seed=2)
    qo, ko = block.rotary(q, k, spec, head_dim=d, positions=torch.tensor(FAR, device=DEV))
    check(qo, q, spec, d, FAR)
    check(ko, k, spec, d, FAR)


@pytest.mark.parametrize("d,rd", [(128, 64), (24, 24)])
@pytest.mark.parametrize("start", [(1 << 32) - 4, -(1 << 32) - 4, (1 << 40) - 2])
def test_counted_positions_across_32_bits(d, rd, start):
    spec, rows, seq = block.Rotary(rd), 21, 9
    q = randn(rows, 2 * d, seed=3)
    qo, _ = block.rotary(q, None, spec, head_dim=d, seq_len=seq, start=start)
    check(qo, q, spec, d, [start + r % seq for r in range(rows)])
