"""Attention on the GPU: norms of its errors per head and 128 rows against the variance of its roundings
(attention_norms.py), over the forms of the call, other scales, and scores of hundreds and thousands in both directions."""
import pytest
import torch

from fuse_b200 import api, block
from tests.attention_norms import check_lse_norms, check_norms, reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(BF16)


def make(rows, kv_rows, hq, hk, d, seed=1):
    return (randn(rows, hq * d, seed=seed), randn(kv_rows, hk * d, seed=seed + 1), randn(kv_rows, hk * d, seed=seed + 2),
            randn(rows, hq * d, seed=seed + 3))


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def run(q, k, v, do, **kw):
    want = reference(q, k, v, do, **kw)
    out, lse = block.attention(q, k, v, return_lse=True, **kw)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    again = block.attention(*leaves, **kw)
    grads = torch.autograd.grad(again, leaves, do)
    torch.cuda.synchronize()
    assert api.read_status()[0] == 0
    check_lse_norms(lse, want["lse"])
    check_norms({"o": out}, want, kw["head_dim"])
    check_norms(dict(zip(("o", "dq", "dk", "dv"), (again.detach(), *grads))), want, kw["head_dim"])


# batch, q_len, kv_len, q_heads, kv_heads
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 128, 128, 1, 1), (2, 127, 127, 2, 1), (1, 129, 129, 3, 3), (1, 256, 256, 6, 2),
                                   (1, 300, 1000, 4, 1), (2, 37, 333, 12, 4), (1, 700, 200, 2, 2), (1, 513, 513, 16, 1), (1, 5, 640, 128, 1),
                                   (1, 3, 200, 160, 1), (1, 1, 5000, 4, 1), (3, 1, 3000, 32, 8), (1, 7, 9000, 3, 1), (1, 40, 6000, 8, 1),
                                   (20, 1, 2000, 32, 8), (1, 1500, 1500, 8, 1), (2, 900, 1100, 6, 2), (3, 2, 700, 20, 4), (2, 1, 900, 7, 1)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(window=200, sinks=150), dict(causal=False)])
def test_norms(shape, d, kw):
    b, ql, kl, hq, hk = shape
    run(*make(b * ql, b * kl, hq, hk, d), head_dim=d, batch=b, **kw)


# a scale of its own goes into the scores, dQ, dK and the join of dK's chunks separately, and through the split over keys
@pytest.mark.parametrize("scale", [0.02, 0.3, 1.0])
@pytest.mark.parametrize("shape", [(1, 300, 300, 2, 2, 128), (1, 1500, 1500, 8, 1, 64), (2, 900, 1100, 6, 2, 128), (1, 2, 5000, 8, 2, 64)])
def test_other_scales(shape, scale):
    b, ql, kl, hq, hk, d = shape
    run(*make(b * ql, b * kl, hq, hk, d, 11), head_dim=d, batch=b, scale=scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
def test_padded_batch(d, window, sinks):
    b, ql, kl = 5, 300, 420
    q, k, v, do = make(b * ql, b * kl, 4, 2, d, 21)
    run(q, k, v, do, head_dim=d, batch=b, window=window, sinks=sinks, q_lengths=i32(300, 0, 1, 129, 200), kv_lengths=i32(420, 17, 0, 128, 100))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("slope", [400.0, -400.0, 3000.0])
def test_scores_of_hundreds_and_thousands_in_both_directions(d, slope):
    """They climb or fall along the keys; the backward makes the weights from them and an lse of that size again."""
    n = 700
    q, k, v, do = make(n, n, 2, 1, d, 31)
    direction = torch.randn(d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    direction = direction / direction.norm()
    q = (0.1 * q.float() + direction.repeat(2) * d ** 0.5).to(BF16)
    k = (k.float() + torch.linspace(-1.0, 1.0, n, device=DEV)[:, None] * slope * direction).to(BF16)
    run(q, k, v, do, head_dim=d)
