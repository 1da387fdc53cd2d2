"""Windowed attention with sinks on the GPU against the formulas in 64 bits (csrc/attention.cuh,
attention_backward.cuh); tolerances: attention_reference.py."""
import pytest
import torch

from fuse_b200 import _native as N
from fuse_b200 import api, block
from tests.attention_reference import attention64, check, check_lse

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def randn(*shape, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)).to(BF16)


def make(rows, kv_rows, hq, hk, d, seed=1, scale=1.0):
    return (randn(rows, hq * d, seed=seed, scale=scale), randn(kv_rows, hk * d, seed=seed + 1), randn(kv_rows, hk * d, seed=seed + 2),
            randn(rows, hq * d, seed=seed + 3))


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def run_all(q, k, v, do, **kw):
    """Forward without gradients (with lse), then forward and backward: every result against 64 bits."""
    want = attention64(q, k, v, do=do, **kw)
    out, lse = block.attention(q, k, v, return_lse=True, **kw)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    again = block.attention(*leaves, **kw)
    dq, dk, dv = torch.autograd.grad(again, leaves, do)
    torch.cuda.synchronize()
    assert api.read_status()[0] == 0
    check({"o": out}, want, ["o"])
    check_lse(lse, want["lse"])
    check({"o": again.detach(), "dq": dq, "dk": dk, "dv": dv}, want, ["o", "dq", "dk", "dv"])
    return out, lse, dq, dk, dv


# batch, q_len, kv_len, q_heads, kv_heads
SHAPES = [(1, 1, 1, 1, 1), (1, 128, 128, 1, 1), (2, 127, 127, 2, 1), (1, 129, 129, 3, 3), (1, 256, 256, 6, 2), (3, 65, 65, 4, 1),
          (1, 300, 1000, 4, 1), (2, 37, 333, 12, 4), (1, 700, 200, 2, 2), (1, 513, 513, 16, 1), (1, 5, 640, 128, 1), (1, 3, 200, 160, 1),
          (2, 1, 130, 8, 8), (1, 200, 0, 2, 1)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
def test_causal(shape, d):
    b, ql, kl, hq, hk = shape
    run_all(*make(b * ql, b * kl, hq, hk, d), head_dim=d, batch=b)


@pytest.mark.parametrize("shape", [(1, 128, 128, 1, 1), (2, 100, 300, 4, 2), (1, 300, 77, 2, 1), (1, 1, 513, 8, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_all_keys_visible(shape, d):
    b, ql, kl, hq, hk = shape
    run_all(*make(b * ql, b * kl, hq, hk, d), head_dim=d, batch=b, causal=False)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (128, 0), (129, 127), (200, 128), (130, 300), (1000, 5), (64, 4000)])
@pytest.mark.parametrize("shape", [(1, 700, 700, 4, 1, 128), (2, 130, 600, 3, 3, 64), (1, 513, 300, 2, 1, 64), (1, 2, 900, 8, 2, 128)])
def test_window_and_sinks(window, sinks, shape):
    b, ql, kl, hq, hk, d = shape
    run_all(*make(b * ql, b * kl, hq, hk, d), head_dim=d, batch=b, window=window, sinks=sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
def test_padded_batch(d, window, sinks):
    b, ql, kl = 5, 300, 420
    q, k, v, do = make(b * ql, b * kl, 4, 2, d)
    ql_, kl_ = i32(300, 0, 1, 129, 200), i32(420, 17, 0, 128, 100)
    for i in range(b):  # whatever lies behind a sequence must not matter
        q[i * ql + int(ql_[i]):(i + 1) * ql] = float("nan")
        do[i * ql + int(ql_[i]):(i + 1) * ql] = float("inf")
        k[i * kl + int(kl_[i]):(i + 1) * kl] = float("nan")
        v[i * kl + int(kl_[i]):(i + 1) * kl] = float("inf")
    out, lse, dq, dk, dv = run_all(q, k, v, do, head_dim=d, batch=b, window=window, sinks=sinks, q_lengths=ql_, kv_lengths=kl_)
    for t, n, lengths in ((out, ql, ql_), (dq, ql, ql_), (dk, kl, kl_), (dv, kl, kl_)):
        for i in range(b):
            assert (t[i * n + int(lengths[i]):(i + 1) * n] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
def test_packed_sequences_in_any_order(d):
    lengths = i32(70, 200, 1, 333, 128)
    starts = i32(700, 10, 211, 300, 850)
    q, k, v, do = make(1000, 1000, 6, 2, d)
    used = torch.zeros(1000, dtype=torch.bool, device=DEV)
    for s, n in zip(starts.tolist(), lengths.tolist()):
        used[s:s + n] = True
    for t in (q, k, v, do):
        t[~used] = float("nan")
    out, *_ = run_all(q, k, v, do, head_dim=d, batch=5, q_len=333, kv_len=333, window=90, sinks=2, q_starts=starts,
                      q_lengths=lengths, kv_starts=starts, kv_lengths=lengths)
    assert (out[~used] == 0).all()


# few query rows against many keys: the keys are split and joined
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", [(1, 1, 5000, 4, 1), (3, 1, 3000, 32, 8), (1, 7, 9000, 3, 1), (2, 2, 2049, 16, 16), (1, 40, 6000, 8, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 130)])
def test_few_rows(shape, d, window, sinks):
    b, ql, kl, hq, hk = shape
    run_all(*make(b * ql, b * kl, hq, hk, d), head_dim=d, batch=b, window=window, sinks=sinks)


def test_few_rows_of_unequal_contexts():
    b, kl, d = 6, 4000, 128
    q, k, v, do = make(b * 2, b * kl, 8, 2, d)
    lengths = i32(4000, 0, 1, 129, 2500, 2)
    for i in range(b):
        k[i * kl + int(lengths[i]):(i + 1) * kl] = float("nan")
        v[i * kl + int(lengths[i]):(i + 1) * kl] = float("nan")
    run_all(q, k, v, do, head_dim=d, batch=b, kv_lengths=lengths)


def test_the_split_path_is_taken():
    p = N.AttentionParams(q_rows=1, kv_rows=8192, batch=1, q_len=1, kv_len=8192, q_heads=8, kv_heads=1, head_dim=128, causal=1, scale=1.0)
    rc, size = api.attention_workspace_size(p)
    assert rc == 0 and size > 0
    p.q_rows = p.q_len = 8192
    p.q_heads = p.kv_heads = 8
    assert api.attention_workspace_size(p) == (0, 0)


@pytest.mark.parametrize("d", [64, 128])
def test_maxima_that_grow_and_far_apart_scores(d):
    """Scores that climb along the keys (every tile raises the reference of the exponent), fall, and span thousands."""
    n = 700
    ramp = torch.linspace(-1.0, 1.0, n, device=DEV)[:, None]
    for slope, seed in ((400.0, 5), (-400.0, 6), (3000.0, 7)):
        q, k, v, do = make(n, n, 2, 1, d, seed)
        direction = torch.randn(d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
        direction = direction / direction.norm()
        q = (0.1 * q.float() + direction.repeat(2) * d ** 0.5).to(BF16)
        k = (k.float() + ramp * slope * direction).to(BF16)
        out, _ = block.attention(q, k, v, head_dim=d, return_lse=True)
        want = attention64(q, k, v, head_dim=d)
        # scores of thousands in FP32 are off by 2^-24 of their size times the products summed: their weights by 2^-24 * s * d
        extra = 2.0 ** -24 * abs(slope) * d
        want["tol_o"] = want["tol_o"] + 4 * extra * v.double().abs().max()
        check({"o": out}, want, ["o"])


def test_gradients_against_differences():
    d, n = 64, 90
    q, k, v, do = make(n, n, 2, 1, d, 21)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    kw = dict(head_dim=d, window=40, sinks=3)
    grads = torch.autograd.grad(block.attention(*leaves, **kw), leaves, do)
    want = attention64(q, k, v, do=do, **kw)
    gen = torch.Generator(device=DEV).manual_seed(22)
    base = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn(base[i].shape, generator=gen, device=DEV, dtype=torch.float64)
        def at(e):
            moved = list(base)
            moved[i] = moved[i] + e * step
            return (attention64(*moved, **kw)["o"] * do.double()).sum()
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        assert (slope - (grads[i].double() * step).sum()).abs() <= (want["tol_" + name] * step.abs()).sum() + 1e-6 * slope.abs() + 1e-6


def test_the_same_every_time():
    q, k, v, do = make(1500, 1500, 8, 2, 128, 31)
    first = None
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = block.attention(*leaves, head_dim=128, window=500, sinks=4)
        got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_views_of_one_packed_tensor_and_a_given_output():
    d, hq, hk, n = 128, 4, 2, 333
    packed = randn(n, (hq + 2 * hk) * d, seed=41)
    q, k, v = packed[:, :hq * d], packed[:, hq * d:(hq + hk) * d], packed[:, (hq + hk) * d:]
    want = block.attention(q.contiguous(), k.contiguous(), v.contiguous(), head_dim=d)
    wide = randn(n, 2 * hq * d, seed=42)
    keep = wide.clone()
    got = block.attention(q, k, v, head_dim=d, out=wide[:, hq * d:])
    assert got.data_ptr() == wide[:, hq * d:].data_ptr()
    assert torch.equal(got, want) and torch.equal(wide[:, :hq * d], keep[:, :hq * d])
    lengths = i32(300)
    wide.copy_(keep)
    block.attention(q, k, v, head_dim=d, out=wide[:, hq * d:], q_lengths=lengths, kv_lengths=lengths)
    assert torch.equal(wide[300:], keep[300:])  # rows behind the sequence as they were
    x = packed.clone().requires_grad_()
    o = block.attention(x[:, :hq * d], x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:], head_dim=d)
    dx, = torch.autograd.grad(o.sum(), x)  # through the views, from an expanded gradient
    ref = attention64(q, k, v, head_dim=d, do=torch.ones_like(want))
    check({"dq": dx[:, :hq * d], "dk": dx[:, hq * d:(hq + hk) * d], "dv": dx[:, (hq + hk) * d:]}, ref, ["dq", "dk", "dv"])


def test_rows_past_31_bits_of_elements():
    rows, width, d = 1_200_000, 2048, 128  # 2.46e9 elements
    kv = torch.zeros(rows, width, dtype=BF16, device=DEV)
    start = rows - 400
    kv[start:] = randn(400, width, seed=51)
    k, v = kv[:, :d], kv[:, d:2 * d]
    q = kv[:, 1024:1024 + 2 * d]
    starts, lengths = i32(start), i32(390)
    out = block.attention(q, k, v, head_dim=d, q_len=390, kv_len=390, q_starts=starts, q_lengths=lengths, kv_starts=starts,
                          kv_lengths=lengths)
    want = attention64(q[start:start + 390], k[start:start + 390], v[start:start + 390], head_dim=d)
    check({"o": out[start:start + 390]}, want, ["o"])
    assert (out[start + 390:] == 0).all() and (out[:1000] == 0).all()


def test_lengths_beyond_the_tensors_touch_nothing_outside():
    q, k, v, _ = make(100, 100, 2, 1, 64, 61)
    guard = torch.zeros(300, 128, dtype=BF16, device=DEV)
    out = guard[100:200]
    for starts, lengths in ((90, 50), (-5, 20), (1000, 30), (50, -3), (0, 2 ** 30)):
        guard.fill_(7.0)
        block.attention(q, k, v, head_dim=64, q_len=100, kv_len=100, q_starts=i32(starts), q_lengths=i32(lengths),
                        kv_starts=i32(starts), kv_lengths=i32(lengths), out=out)
        torch.cuda.synchronize()
        assert (guard[:100] == 7).all() and (guard[200:] == 7).all()


def test_captured_on_side_streams_and_with_eager_graphs_alive():
    q, k, v, do = make(260, 260, 4, 2, 64, 71)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = block.attention(*leaves, head_dim=64, window=50, sinks=1)
        grads = torch.autograd.grad(o, leaves, do)
    torch.cuda.current_stream().wait_stream(side)
    want = attention64(q, k, v, do=do, head_dim=64, window=50, sinks=1)
    check(dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads))), want, ["o", "dq", "dk", "dv"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = block.attention(*leaves, head_dim=64, window=50, sinks=1)
        grads = torch.autograd.grad(o, leaves, do)
    fresh = make(260, 260, 4, 2, 64, 81)
    with torch.no_grad():
        for t, f in zip(leaves, fresh):
            t.copy_(f)
    do.copy_(fresh[3])
    graph.replay()
    torch.cuda.synchronize()
    want = attention64(*fresh[:3], do=fresh[3], head_dim=64, window=50, sinks=1)
    check(dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads))), want, ["o", "dq", "dk", "dv"])


def test_two_captured_graphs_with_splits_do_not_share_memory():
    q, k, v, _ = make(1, 6000, 8, 1, 128, 91)
    q2, k2, v2, _ = make(1, 6000, 8, 1, 128, 95)
    graphs, outs = [], []
    for args in ((q, k, v), (q2, k2, v2)):
        block.attention(*args, head_dim=128)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(block.attention(*args, head_dim=128))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, args in zip(outs, ((q, k, v), (q2, k2, v2))):
        check({"o": out}, attention64(*args, head_dim=128), ["o"])


def test_refusals():
    q, k, v, do = make(64, 64, 4, 2, 64, 101)
    for call in (lambda: block.attention(q, k, v, head_dim=48), lambda: block.attention(q, k, v[:32], head_dim=64),
                 lambda: block.attention(q, k, v, head_dim=64, batch=3), lambda: block.attention(q, k, v, head_dim=64, window=-1),
                 lambda: block.attention(q, k, v, head_dim=64, causal=False, window=8),
                 lambda: block.attention(q, k, v, head_dim=64, q_lengths=torch.zeros(1, device=DEV)),
                 lambda: block.attention(q, k, v, head_dim=64, kv_starts=i32(0, 0)),
                 lambda: block.attention(q.float(), k, v, head_dim=64), lambda: block.attention(q[:, :192], k, v, head_dim=64)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: block.attention(q, k, v, head_dim=32), lambda: block.attention(q, k, v, head_dim=64, scale=-1.0),
                 lambda: block.attention(q, k, v, head_dim=64, kv_len=65),
                 lambda: block.attention(q.clone().requires_grad_(), k, v, head_dim=64, out=torch.empty_like(q))):
        with pytest.raises(RuntimeError):
            call()


# key tiles that many query tiles see are made in chunks: all (causal, few KV heads), or those with sinks
@pytest.mark.parametrize("kw", [dict(), dict(window=200, sinks=150), dict(window=40, sinks=1), dict(causal=False), dict(window=900, sinks=0)])
@pytest.mark.parametrize("shape", [(1, 1500, 1500, 8, 1, 64), (2, 900, 1100, 6, 2, 128)])
def test_key_gradients_in_chunks(kw, shape):
    b, ql, kl, hq, hk, d = shape
    run_all(*make(b * ql, b * kl, hq, hk, d, 111), head_dim=d, batch=b, **kw)


def test_workspace_of_a_long_context_stays_small():
    p = N.AttentionBackwardParams(forward=N.AttentionParams(
        q_rows=1 << 19, kv_rows=1 << 19, batch=1, q_len=1 << 19, kv_len=1 << 19, q_heads=8, kv_heads=1, head_dim=128, causal=1,
        window=4096, sinks=4, scale=1.0))
    rc, size = api.attention_backward_workspace_size(p)
    assert rc == 0 and size < 1 << 27
    p.forward.window = 0
    rc, size = api.attention_backward_workspace_size(p)
    assert rc == 0 and size < 1 << 27
    p.forward.q_len = p.forward.kv_len = p.forward.q_rows = p.forward.kv_rows = 25600
    p.forward.window = 128
    rc, size = api.attention_backward_workspace_size(p)
    assert rc == 0 and size < 1 << 28


def test_shared_keys_without_gradients():
    q, k, v, _ = make(3 * 20, 500, 4, 2, 64, 121)
    out = block.attention(q, k, v, head_dim=64, batch=3, kv_len=500, kv_starts=i32(0, 0, 100), kv_lengths=i32(500, 300, 300))
    for i, (s, n) in enumerate(((0, 500), (0, 300), (100, 300))):
        want = attention64(q[20 * i:20 * i + 20], k[s:s + n], v[s:s + n], head_dim=64)
        check({"o": out[20 * i:20 * i + 20]}, want, ["o"])


def test_no_queries_and_no_keys():
    q, k, v, _ = make(0, 64, 2, 1, 64, 131)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = block.attention(*leaves, head_dim=64)
    assert out.shape == (0, 128)
    dq, dk, dv = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert dq.shape == (0, 128) and (dk == 0).all() and (dv == 0).all()
    q, k, v, do = make(40, 64, 2, 1, 64, 132)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out, lse = block.attention(*leaves, head_dim=64, kv_lengths=i32(0), return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all()
    assert all((g == 0).all() for g in torch.autograd.grad(out, leaves, do))
