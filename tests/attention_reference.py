"""Windowed attention with sinks in 64 bits, one sequence and head at a time, with the gradients and the sizes that the
tolerances of the GPU tests are made of.

Tolerances (u = 2^-8, half a BF16 step relative to the value; a row's P sums to 1).
  o:  its own rounding u |o|, and the rounding of every weight before the product, u P|V|.
  dv: u |dv| and, by the same rounding, u P^T |dO|.
  dS: rounded, u |dS|; D = rowsum(dO O) carries O's error, e = |dO| . tol(o), and enters as P e.
  dq: u |dq| + scale (u |dS| + P e) |K|;   dk: u |dk| + scale (u |dS| + P e)^T |Q|.
FP32 adds, to scores, dP and sums of a few thousand terms of BF16 products, well below 2^-11 of the sizes summed (2^-24
times fewer than 2^12 terms, times a score of at most 2): the u of every product of weights is taken as 2^-8 + 2^-11, and
dP's own error as 2^-11 P (|dO| |V|^T) beside P e."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -8
W = U + 2.0 ** -11


def attention64(q, k, v, *, head_dim, batch=1, causal=True, window=0, sinks=0, scale=None, q_len=None, kv_len=None,
                q_starts=None, q_lengths=None, kv_starts=None, kv_lengths=None, do=None):
    """Dict of o, lse [q_heads, rows] and, with `do`, dq, dk, dv; for each tensor a tolerance under "tol_...".  Rows of
    no sequence: zeros (lse -inf)."""
    d, f64 = head_dim, torch.float64
    hq, hk = q.shape[1] // d, k.shape[1] // d
    scale = d ** -0.5 if scale is None else scale
    q_len = q.shape[0] // batch if q_len is None else q_len
    kv_len = k.shape[0] // batch if kv_len is None else kv_len
    names = ["o", "dq", "dk", "dv"]
    out = {n: torch.zeros((q if n in ("o", "dq") else k).shape, dtype=f64, device=q.device) for n in names}
    out.update({"tol_" + n: torch.zeros_like(out[n]) for n in names})
    out["lse"] = torch.full((hq, q.shape[0]), -math.inf, dtype=f64, device=q.device)

    def rows(starts, lengths, b, most):
        first = int(starts[b]) if starts is not None else b * most
        return slice(first, first + (int(lengths[b]) if lengths is not None else most))

    for b in range(batch):
        rq, rk = rows(q_starts, q_lengths, b, q_len), rows(kv_starts, kv_lengths, b, kv_len)
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        pos = torch.arange(nq, device=q.device)[:, None] + (nk - nq)
        key = torch.arange(nk, device=q.device)[None, :]
        seen = key <= pos if causal else torch.ones((nq, nk), dtype=torch.bool, device=q.device)
        if causal and window:
            seen = seen & ((pos - key < window) | (key < sinks))
        for h in range(hq):
            g = h // (hq // hk)
            cq, ck = slice(h * d, (h + 1) * d), slice(g * d, (g + 1) * d)
            Q, K, V = q[rq, cq].to(f64), k[rk, ck].to(f64), v[rk, ck].to(f64)
            s = ((Q @ K.T) * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, dim=1, keepdim=True) if nk else torch.full((nq, 1), -math.inf, dtype=f64, device=q.device)
            p = torch.where(seen, torch.exp(s - lse), torch.zeros_like(s))
            o = p @ V
            tol_o = U * o.abs() + W * (p @ V.abs())
            out["o"][rq, cq], out["tol_o"][rq, cq], out["lse"][h, rq] = o, tol_o, lse[:, 0]
            if do is None:
                continue
            G = do[rq, cq].to(f64)
            dp = G @ V.T
            ds = p * (dp - (G * o).sum(1, keepdim=True))
            e = W * ds.abs() + p * ((G.abs() * tol_o).sum(1, keepdim=True) + 2.0 ** -11 * (G.abs() @ V.abs().T))
            out["dq"][rq, cq] = scale * ds @ K
            out["tol_dq"][rq, cq] = U * out["dq"][rq, cq].abs() + scale * e @ K.abs()
            out["dk"][rk, ck] += scale * ds.T @ Q
            out["tol_dk"][rk, ck] += scale * e.T @ Q.abs()
            out["dv"][rk, ck] += p.T @ G
            out["tol_dv"][rk, ck] += W * p.T @ G.abs()
    for n in ("dk", "dv"):
        out["tol_" + n] += U * out[n].abs()
    return out


def check(got, want, names):
    for n in names:
        diff, tol = (got[n].double() - want[n]).abs(), want["tol_" + n] + 2.0 ** -133
        bad = ~(diff <= tol)
        assert not bad.any(), (n, int(bad.sum()), float(diff[bad].max()), float((diff / tol).nan_to_num(math.inf).max()))


def check_lse(got, want):
    """Within 2^-11 of a score's size, by the same count of FP32 roundings; -inf where nothing is seen."""
    empty = torch.isinf(want)
    assert torch.equal(torch.isinf(got), empty) and (got[empty] < 0).all()
    assert ((got.double() - want)[~empty].abs() <= 2.0 ** -11 * (1.0 + want[~empty].abs())).all()
