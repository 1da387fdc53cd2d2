"""Attention on the GPU: norms of its errors per head and 128 rows against the variance of its roundings
(attention_norms.py), over the forms of the call, other scales, and scores of hundreds and thousands in both directions."""
import pytest
import torch

from fuse_b200 import _native as N
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


# Where a row's weight lies on few keys (short sequences, short windows, scores far apart), dS = P (dP - D) is small beside D, and
# what D is off by stands out.  Three independent roundings make the gradients: dS's, their own, and P's, which D carries through
# the output.  A BF16 rounding is half a step at most, evenly spread; over evenly spread logarithms of the value its root mean square is
# 2^-7 / sqrt(12) * sqrt(0.75 / (2 ln 2)) = 0.00166.  sqrt(3) of it, and a quarter more for chance in a few hundred values.
BOUND = 3 ** 0.5 * 0.00166 * 1.25


@pytest.mark.parametrize("n,window,sharp", [(2, 0, 1.0), (3, 0, 1.0), (6, 0, 1.0), (16, 0, 1.0), (1024, 2, 1.0), (1024, 4, 1.0), (64, 0, 8.0),
                                            (1024, 0, 8.0), (64, 0, 16.0), (1024, 0, 16.0)])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_rows_whose_weight_lies_on_few_keys(n, window, sharp, d):
    batch = 8 if n <= 64 else 1
    q, k, v, do = make(batch * n, batch * n, 4, 2, d, 41)
    q = (q.float() * sharp).to(BF16)
    kw = dict(head_dim=d, batch=batch, window=window)
    want = reference(q, k, v, do, **kw)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(block.attention(*leaves, **kw), leaves, do)
    for name, got in zip(("dq", "dk", "dv"), grads):
        value = want[name][0]
        assert float((got.double() - value).norm() / value.norm()) <= BOUND, name


def record(q, k, v, out, lse, hq, hk, d, rest=None, **kw):
    p = N.AttentionParams(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), output=out.data_ptr(), lse=lse.data_ptr(), q_stride=-1, k_stride=-1,
                          v_stride=-1, output_stride=out.stride(0), q_rows=q.shape[0], kv_rows=k.shape[0], batch=1, q_len=q.shape[0],
                          kv_len=k.shape[0], q_heads=hq, kv_heads=hk, head_dim=d, causal=0, scale=d ** -0.5,
                          output_rest=None if rest is None else rest.data_ptr(), **kw)
    rc, size = api.attention_workspace_size(p)
    work = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = work.data_ptr(), size
    return rc, p, work


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len,kv_len", [(300, 700), (2, 5000)])  # the second is split and joined
def test_output_and_its_rest_hold_sixteen_bits(q_len, kv_len, d):
    """Equal scores: every weight is 1, the output a mean, exact but for FP32's additions (2^-24 of the sizes each)."""
    q, k, v, _ = make(q_len, kv_len, 4, 2, d, 51)
    k.zero_()
    wide, rest, lse = torch.zeros(q_len, 8 * d, dtype=BF16, device=DEV), torch.zeros(q_len + 1, 4 * d, dtype=torch.int8, device=DEV), torch.empty(4, q_len, device=DEV)
    out = wide[:, 4 * d:]
    rc, p, work = record(q, k, v, out, lse, 4, 2, d, rest)
    assert rc == 0 and api.launch_attention(p) == 0
    torch.cuda.synchronize()
    mean = v.double().view(kv_len, 2, 1, d).mean(0).expand(2, 2, d).reshape(1, -1)
    size = v.double().abs().view(kv_len, 2, 1, d).mean(0).expand(2, 2, d).reshape(1, -1)
    both = ((out.contiguous().view(torch.int16).int() << 16) + (rest[:q_len].int() << 8)).view(torch.float32).double()
    # half a unit of the byte: 2^7 of 2^24 at most; the sum in steps of sixteen and the joining of parts
    assert ((both - mean).abs() <= mean.abs() * 2.0 ** -16 + size * (kv_len / 16 + 16) * 2.0 ** -24).all()
    assert ((out.double() - mean).abs() <= mean.abs() * 2.0 ** -8 + size * (kv_len / 16 + 16) * 2.0 ** -24).all()
    assert (rest[q_len] == 0).all() and (wide[:, :4 * d] == 0).all() and (rest[:q_len] != 0).any()
    # the output itself does not depend on whether the rest is asked for
    again = torch.zeros_like(wide)
    rc, p, work = record(q, k, v, again[:, 4 * d:], lse, 4, 2, d)
    assert rc == 0 and api.launch_attention(p) == 0
    torch.cuda.synchronize()
    assert torch.equal(again, wide)


def test_rest_of_a_padded_batch_and_of_numbers_that_are_none():
    d = 64
    q, k, v, _ = make(300, 300, 1, 1, d, 61)
    v[:, 0], v[5, 1], q[7] = float("inf"), float("nan"), float("nan")
    out, rest, lse = torch.zeros(300, d, dtype=BF16, device=DEV), torch.full((300, d), 77, dtype=torch.int8, device=DEV), torch.empty(1, 300, device=DEV)
    lengths = i32(200)
    rc, p, work = record(q, k, v, out, lse, 1, 1, d, rest, q_lengths=lengths.data_ptr(), kv_lengths=lengths.data_ptr())
    assert rc == 0 and api.launch_attention(p) == 0
    torch.cuda.synchronize()
    assert (rest[200:] == 77).all() and (out[200:] == 0).all()  # rows of no sequence as they were
    both = ((out[:200].view(torch.int16).int() << 16) + (rest[:200].int() << 8)).view(torch.float32)
    assert torch.equal(torch.isnan(both), torch.isnan(out[:200])) and torch.equal(torch.isinf(both), torch.isinf(out[:200]))
    assert torch.isinf(out[:7, 0]).all() and torch.isnan(out[:200, 1]).all() and torch.isnan(out[7]).all()


def test_backward_without_the_rest():
    """The record's output_rest may be NULL in the backward: D then comes from the rounded output, within the bounds for that."""
    d, n = 64, 300
    q, k, v, do = make(n, n, 4, 2, d, 71)
    want = reference(q, k, v, do, head_dim=d, causal=False)
    out, lse = torch.empty_like(q), torch.empty(4, n, device=DEV)
    rc, p, work = record(q, k, v, out, lse, 4, 2, d)
    assert rc == 0 and api.launch_attention(p) == 0
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    g = N.AttentionBackwardParams(forward=p, grad_output=do.data_ptr(), grad_q=dq.data_ptr(), grad_k=dk.data_ptr(), grad_v=dv.data_ptr(),
                                  grad_output_stride=-1, grad_q_stride=-1, grad_k_stride=-1, grad_v_stride=-1)
    rc, size = api.attention_backward_workspace_size(g)
    space = torch.empty(size, dtype=torch.uint8, device=DEV)
    g.workspace, g.workspace_bytes = space.data_ptr(), size
    assert rc == 0 and api.launch_attention_backward(g) == 0
    torch.cuda.synchronize()
    check_norms({"dq": dq, "dk": dk, "dv": dv}, want, d)
