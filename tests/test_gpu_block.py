"""The block operators in a row with the fused projections, as a layer uses them, against native torch autograd in FP32 and
against the oracle on the quantised path."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from fuse_b200 import block

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16 = torch.bfloat16
SPEC = dict(rotary_dim=128, theta=10000.0, scaling="wavelength", factor=4.0, original_context=64)


def reference_rotary(x, heads, d, seq):
    f, m = block.Rotary(**SPEC).frequencies()
    angle = (torch.arange(x.shape[0], device=DEV) % seq).double()[:, None] * torch.tensor(f, dtype=torch.float64, device=DEV)
    c, s = (torch.cos(angle) * m).float()[:, None], (torch.sin(angle) * m).float()[:, None]
    x = x.view(-1, heads, d)
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat((a * c - b * s, a * s + b * c), -1).view(x.shape[0], -1)


def reference_attention(q, k, v, batch, hq, hk, d, window, sinks):
    n = q.shape[0] // batch
    q = q.view(batch, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    k, v = (t.view(batch, n, hk, 1, d).permute(0, 2, 3, 1, 4) for t in (k, v))
    i, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    p = torch.softmax((q @ k.transpose(-1, -2) * d ** -0.5).masked_fill(~seen, -torch.inf), -1)
    return (p @ v).permute(0, 3, 1, 2, 4).reshape(batch * n, -1)


def test_layer_of_norm_projections_rotary_and_attention():
    from fuse_b200.autograd import UlyssesProjections
    from fuse_b200.world import World
    batch, seq, hidden, hq, hk, d, window, sinks = 2, 256, 512, 4, 2, 128, 100, 4
    gen = torch.Generator(device=DEV).manual_seed(7)
    def rand(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=gen, device=DEV)).to(BF16)
    rows, width = batch * seq, (hq + 2 * hk) * d
    x, stream = rand(rows, hidden), rand(rows, hidden)
    gamma, w_qkv, w_o = (1 + rand(hidden, scale=0.1).float()).to(BF16), rand(width, hidden, scale=0.05), rand(hidden, hq * d, scale=0.05)
    dy, dh = rand(rows, hidden), rand(rows, hidden)
    proj = UlyssesProjections(World(0, 1, 0), batch=batch, seq_local=seq, hidden=hidden, q_heads=hq, kv_heads=hk, head_dim=d,
                              tag="layer")

    def ours(leaves):
        x, stream, gamma, w_qkv, w_o = leaves
        y, h = block.rms_norm(x, gamma, stream)
        q, k, v = proj.qkv(y, w_qkv)
        return proj.oproj(proj.attention(q, k, v, rotary=block.Rotary(**SPEC), window=window, sinks=sinks), w_o), h

    def reference(leaves):
        x, stream, gamma, w_qkv, w_o = leaves
        h = x + stream
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * gamma
        q, k, v = F.linear(y, w_qkv).split([hq * d, hk * d, hk * d], dim=1)
        q, k = reference_rotary(q, hq, d, seq), reference_rotary(k, hk, d, seq)
        return F.linear(reference_attention(q, k, v, batch, hq, hk, d, window, sinks), w_o), h

    source = (x, stream, gamma, w_qkv, w_o)
    want_leaves = [t.float().requires_grad_() for t in source]
    want = reference(want_leaves)
    want = (*want, *torch.autograd.grad(want, want_leaves, (dy.float(), dh.float())))
    for _ in range(2):  # twice: epochs advance, buffers are reused
        leaves = [t.clone().requires_grad_() for t in source]
        got = ours(leaves)
        got = (*got, *torch.autograd.grad(got, leaves, (dy, dh)))
        for name, a, b in zip(("y", "h", "dx", "dstream", "dgamma", "dw_qkv", "dw_o"), got, want):
            # some ten BF16 roundings of 2^-9 (root mean square 2^-9 / sqrt 3 each) between an input and the furthest output
            rel = (a.float() - b).norm() / b.norm()
            assert rel <= 10 * 2.0 ** -9, (name, float(rel))
    with torch.no_grad():  # without gradients the attention writes where the output projection reads
        y, h = block.rms_norm(x, gamma, stream)
        q, k, v = proj.qkv(y, w_qkv)
        a = proj.attention(q, k, v, rotary=block.Rotary(**SPEC), window=window, sinks=sinks, out=proj.attention_buffer())
        assert torch.equal(proj.oproj(a, w_o), got[0])


def test_norm_feeds_the_mxfp8_projection():
    from oracle import oracle as O
    from tests import harness as H
    m, hidden, n = 256, 512, 384
    gen = torch.Generator(device=DEV).manual_seed(9)
    x, res = (torch.randn(m, hidden, generator=gen, device=DEV).to(BF16) for _ in range(2))
    gamma = (1 + 0.2 * torch.randn(hidden, generator=gen, device=DEV)).to(BF16)
    w = H.to_bits((0.05 * torch.randn(n, hidden, generator=gen, device=DEV)).to(BF16))
    h, data, scales = block.rms_norm_mxfp8(x, gamma, res)
    y, _ = block.rms_norm(x, gamma, res)
    data, scales = data.cpu().numpy(), scales.cpu().numpy()
    want_data, want_scales = O.mxfp8_quantize(H.to_bits(y))
    assert np.array_equal(data, want_data) and np.array_equal(scales, want_scales)
    out, _, _ = H.qkv_forward_mxfp8(1, 1, m, 1, 1, 8, [data], [scales], w, mode="compute")
    wq, wsf = O.mxfp8_quantize(w)
    ok, worst, bad = O.within_tolerance(out[0], O.gemm_mxfp8(data, scales, wq, wsf))
    assert ok, (worst, bad)
