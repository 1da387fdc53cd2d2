"""Attention at the ends of its ranges.  Positions far along a long cache: gradients of a window and sinks past 16 million keys, where a position
times the heads of a tile no longer fits 31 bits (csrc/attention_backward.cuh).  What lies between the sinks and the window is
seen by nobody, so the same tensors without it give the same results; tolerances: attention_reference.py."""
import pytest
import torch

from fuse_b200 import api, block
from tests.attention_reference import attention64, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.mark.parametrize("window,sinks", [(256, 4), (100, 130)])
def test_sinks_and_window_far_apart(window, sinks):
    d, hq, q_len, head, tail = 64, 128, 4, 256, 512
    kv_len = (1 << 24) + 2048
    gen = torch.Generator(device=DEV).manual_seed(5)

    def randn(rows, width):
        return torch.randn(rows, width, generator=gen, device=DEV).to(BF16)

    q, do = randn(q_len, hq * d), randn(q_len, hq * d)
    ends = [randn(head + tail, d) for _ in range(2)]
    far = []
    for t in ends:
        whole = torch.zeros(kv_len, d, dtype=BF16, device=DEV)
        whole[:head], whole[kv_len - tail:] = t[:head], t[head:]
        far.append(whole)
    want = attention64(q, *ends, head_dim=d, window=window, sinks=sinks, do=do)
    leaves = [t.requires_grad_() for t in (q, *far)]
    out = block.attention(*leaves, head_dim=d, window=window, sinks=sinks)
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    torch.cuda.synchronize()
    assert api.read_status()[0] == 0
    assert not dk[sinks:kv_len - tail].any() and not dv[sinks:kv_len - tail].any()  # seen by nobody
    got = {"o": out.detach(), "dq": dq, **{n: torch.cat((t[:head], t[kv_len - tail:])) for n, t in (("dk", dk), ("dv", dv))}}
    check(got, want, ["o", "dq", "dk", "dv"])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 129, 300, 600])
def test_a_window_that_limits_nothing_changes_nothing(n, d):
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v, do = (torch.randn(n, d, generator=gen, device=DEV).to(BF16) for _ in range(4))
    results = []
    for kw in (dict(), dict(window=n), dict(window=(1 << 31) - 1, sinks=(1 << 31) - 1), dict(window=n + 1, sinks=5), dict(sinks=7)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = block.attention(*leaves, head_dim=d, **kw)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, do)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
