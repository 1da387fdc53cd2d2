"""The accuracy check of the attention tests, on the CPU: it passes results rounded as the kernels round them and fails results
that lack a term of the gradients, a tile of keys or a chunk of queries."""
import pytest
import torch

from tests.attention_norms import check_lse_norms, check_norms, ratios, reference

BF16 = torch.bfloat16
GRADS = ("o", "dq", "dk", "dv")


def inputs(rows, kv_rows, hq, hk, d, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(r, w * d, generator=gen).to(BF16) for r, w in ((rows, hq), (kv_rows, hk), (kv_rows, hk), (rows, hq))]


def rounded(q, k, v, do, head_dim, **kw):
    """The same with the weights and dS rounded to BF16 for their products, D from the rounded output, as the kernels do it."""
    d, (hq, hk) = head_dim, (q.shape[1] // head_dim, k.shape[1] // head_dim)
    scale = kw.get("scale") or d ** -0.5
    out = {n: torch.zeros(t.shape, dtype=torch.float64) for n, t in zip(GRADS, (q, q, k, v))}
    nq, nk = q.shape[0], k.shape[0]
    distance = torch.arange(nq)[:, None] + (nk - nq) - torch.arange(nk)[None]
    sees = distance >= 0 if kw.get("causal", True) else torch.ones_like(distance, dtype=torch.bool)
    for h in range(hq):
        cq, ck = slice(h * d, h * d + d), slice(h // (hq // hk) * d, h // (hq // hk) * d + d)
        Q, K, V, G = (t[:, c].double() for t, c in ((q, cq), (k, ck), (v, ck), (do, cq)))
        s = (scale * Q @ K.T).masked_fill(~sees, -torch.inf)
        top = s.amax(1, keepdim=True)
        w = torch.exp(s - top)
        total = w.sum(1, keepdim=True)
        o = (w.to(BF16).double() @ V / total).to(BF16).double()
        P = w / total
        dS = (P * (G @ V.T - (G * o).sum(1, keepdim=True))).to(BF16).double()
        out["o"][:, cq], out["dq"][:, cq] = o, scale * dS @ K
        out["dk"][:, ck] += scale * dS.T @ Q
        out["dv"][:, ck] += P.to(BF16).double().T @ G
    return {n: t.to(BF16) for n, t in out.items()}


CASES = [((384, 384, 4, 1, 64), dict()), ((1500, 1500, 8, 1, 64), dict(causal=False)), ((40, 6000, 8, 1, 128), dict()),
         ((7, 5000, 3, 1, 64), dict()), ((1, 1, 1, 1, 64), dict()), ((300, 500, 2, 2, 128), dict(scale=0.02))]


@pytest.mark.parametrize("shape,kw", CASES)
def test_what_the_kernels_round_passes(shape, kw):
    tensors, d = inputs(*shape), shape[-1]
    check_norms(rounded(*tensors, head_dim=d, **kw), reference(*tensors, head_dim=d, **kw), d)


@pytest.mark.parametrize("shape,kw", [c for c in CASES if c[0][1] > 1])
def test_wrong_gradients_fail(shape, kw):
    tensors, d, nk, nq = inputs(*shape), shape[-1], shape[1], shape[0]
    want = reference(*tensors, head_dim=d, **kw)
    tile, token = nk // 2, nq // 2
    mistakes = {"no D": lambda i, j, P, dP, D: P * dP,
                "a tile of keys lost": lambda i, j, P, dP, D: P * (dP - D) * ~((j >= tile) & (j < tile + 128)),
                "queries lost": lambda i, j, P, dP, D: P * (dP - D) * ~((i >= token) & (i < token + 16)),
                "D of the next row": lambda i, j, P, dP, D: P * (dP - D.roll(1, 0)) if nq > 1 else P * dP}
    for what, wrong in mistakes.items():
        got = reference(*tensors, head_dim=d, wrong=wrong, **kw)
        for name in ("dq", "dk"):
            worst = float(ratios(got[name][0].to(BF16), want[name], d).max())
            assert worst > 1.0, (what, name, worst)


def test_sums_of_rounded_weights_fail():
    q, k, v, do = inputs(64, 300, 2, 1, 64)
    want = reference(q, k, v, do, head_dim=64)["lse"]
    check_lse_norms(want[0].float(), want)
    with pytest.raises(AssertionError):
        check_lse_norms((want[0] + 1e-4).float(), want)
