"""Windowed attention with sinks in 64 bits, with the size of the rounding errors that its outputs should have together: for
every head and every 128 rows the norm of the error is held against the root of the summed variances.  Single elements may
be as wrong as a gradient is large and still lie within a bound that adds worst cases; a lost term does not hide in a norm.

A rounding to BF16 is off by at most 2^-8 of the value and, as errors spread evenly up to that, by R = 2^-8 / sqrt(3) of it
in the root mean square.  Roundings of different values are independent; their variances add.
  o:  its own, R^2 o^2, and those of the weights, R^2 P^2 V^2.
  dv: R^2 dv^2 + R^2 (P^2)^T dO^2.
  D = rowsum(dO O) carries O's error: its variance is vD = sum dO^2 var(o), one number for all keys of a row.
  dq: R^2 dq^2 + scale^2 (R^2 dS^2 K^2 + vD (P K)^2);  dk: R^2 dk^2 + scale^2 (R^2 (dS^2)^T Q^2 + (P^2 vD)^T Q^2).
FP32, taken as errors of one sign: a score's sum of products goes through at most eight steps of sixteen, each within 2^-24
of the sizes summed, and is scaled by a rounded factor in a rounded product: below 2^-20 scale |Q| |K|^T; lse, its conversion to base 2 and the
factor for it are three roundings, below 2^-22 of it; both move a weight by that part of it (E), and dP is 2^-20 |dO| |V|^T off.  D is then off by |dO| (E P |V|) as well.
The range: ex2.approx.ftz gives 0 below 2^-126, so a weight, and the dS made of it, may also be off by TINY = 2^-126.  (With scores that
fall by 800 over 700 keys, keys 128 to 383 have weights of e^-146 = 2^-211 down to 2^-631 in 64 bits and 0 in FP32: all of a
group's gradient is lost, and rightly.)

FACTOR = 3 roots are allowed.  The fewest independent errors a norm may rest on is one (D of a single row), a sum of 64 and
more terms and so near normal; real mantissas are spread, which makes its deviation 0.74 of the R above: four of its own."""
from __future__ import annotations

import math

import torch

R = 2.0 ** -8 / math.sqrt(3.0)
FACTOR = 3.0
F64 = torch.float64
GROUP = 128
TINY = 2.0 ** -126


def _spans(starts, lengths, batch, most):
    for b in range(batch):
        first = int(starts[b]) if starts is not None else b * most
        yield slice(first, first + (int(lengths[b]) if lengths is not None else most))


def reference(q, k, v, do, *, head_dim, batch=1, causal=True, window=0, sinks=0, scale=None, q_len=None, kv_len=None,
              q_starts=None, q_lengths=None, kv_starts=None, kv_lengths=None, wrong=None):
    """name -> (value, variance, one-sided error) for o, dq, dk, dv, and lse -> (value, bound).  `wrong(i, j, P, dP, D)`, for
    tests of the check itself, returns what takes the place of dS of query i and key j (index tensors)."""
    d = head_dim
    hq, hk = q.shape[1] // d, k.shape[1] // d
    scale = d ** -0.5 if scale is None else scale
    zeros = {n: torch.zeros((q if n in ("o", "dq") else k).shape, dtype=F64, device=q.device) for n in ("o", "dq", "dk", "dv")}
    out = {n: (z, z.clone(), z.clone()) for n, z in zeros.items()}
    lse_value = torch.full((hq, q.shape[0]), -math.inf, dtype=F64, device=q.device)
    lse_bound = torch.zeros_like(lse_value)
    q_len, kv_len = q.shape[0] // batch if q_len is None else q_len, k.shape[0] // batch if kv_len is None else kv_len
    for rq, rk in zip(_spans(q_starts, q_lengths, batch, q_len), _spans(kv_starts, kv_lengths, batch, kv_len)):
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if not nq or not nk:
            continue
        i, j = torch.arange(nq, device=q.device)[:, None], torch.arange(nk, device=q.device)[None]
        distance = i + (nk - nq) - j
        sees = distance >= 0 if causal else torch.ones_like(distance, dtype=torch.bool)
        if causal and window:
            sees = sees & ((distance < window) | (j < sinks))
        for h in range(hq):
            kv = h // (hq // hk)
            cq, ck = slice(h * d, h * d + d), slice(kv * d, kv * d + d)
            Q, K, V, G = (t[r, c].to(F64) for t, r, c in ((q, rq, cq), (k, rk, ck), (v, rk, ck), (do, rq, cq)))
            s = (scale * (Q @ K.T)).masked_fill(~sees, -math.inf)
            top = s.amax(1, keepdim=True).clamp_min(-1e300)
            w = torch.exp(s - top)
            total = w.sum(1, keepdim=True)
            P = w / total.clamp_min(1e-300)
            lse = torch.where(total > 0, top + torch.log(total.clamp_min(1e-300)), torch.full_like(top, -math.inf))
            size = 2.0 ** -20 * scale * (Q.abs() @ K.abs().T)
            E = (size + 2.0 ** -22 * torch.where(total > 0, lse.abs(), torch.zeros_like(lse))) * P + TINY * sees  # of a weight
            o = P @ V
            var_o = R * R * (o * o + (P * P) @ (V * V))
            one_o = E @ V.abs()
            dP = G @ V.T
            D = (G * o).sum(1, keepdim=True)
            dS = P * (dP - D)
            if wrong is not None:
                dS = wrong(i, j, P, dP, D)
            vD = (G * G * var_o).sum(1, keepdim=True)
            one_D = (G.abs() * one_o).sum(1, keepdim=True)
            one_dS = TINY * sees + E * (dP - D).abs() + P * (one_D + 2.0 ** -20 * (G.abs() @ V.abs().T))
            sd2 = scale * scale
            terms = {"o": (rq, cq, o, var_o, one_o),
                     "dq": (rq, cq, scale * dS @ K, sd2 * (R * R * (dS * dS) @ (K * K) + vD * (P @ K) ** 2), scale * one_dS @ K.abs()),
                     "dk": (rk, ck, scale * dS.T @ Q, sd2 * (R * R * dS * dS + P * P * vD).T @ (Q * Q), scale * one_dS.T @ Q.abs()),
                     "dv": (rk, ck, P.T @ G, R * R * (P * P).T @ (G * G), E.T @ G.abs())}
            for name, (rows, columns, *values) in terms.items():
                for to, value in zip(out[name], values):
                    to[rows, columns] += value
            lse_value[h, rq] = lse[:, 0]
            # the sum: exponentials within 2^-22, twenty additions a key tile and one a tile, each 2^-24 (all of one sign);
            # joined parts go through as much again; the logarithm and its scaling a few roundings of the result
            lse_bound[h, rq] = (size.masked_fill(~sees, 0.0).amax(1) + 2.0 ** -22 * lse[:, 0].abs().nan_to_num(posinf=0.0) +
                                2.0 ** -20 + (40 + nk / 64) * 2.0 ** -24)
    for name in ("dq", "dk", "dv"):  # their own rounding
        out[name][1].add_(R * R * out[name][0] ** 2)
    return {**out, "lse": (lse_value, lse_bound)}


def ratios(got, want, head_dim):
    """Norm of the error over what is allowed, [groups of rows, heads]."""
    value, variance, one = want
    rows, width = value.shape
    pad = -rows % GROUP

    def summed(x):  # of squares, by group
        x = torch.nn.functional.pad(x, (0, 0, 0, pad)).view(-1, GROUP, width // head_dim, head_dim)
        return x.sum((1, 3))

    error = summed((got.to(F64) - value) ** 2).sqrt()
    allowed = FACTOR * summed(variance).sqrt() + summed(one * one).sqrt()
    return torch.where(error == 0, torch.zeros_like(error), error / allowed)


def check_norms(got, want, head_dim):
    for name, tensor in got.items():
        worst = ratios(tensor, want[name], head_dim)
        assert bool((worst <= 1.0).all()), (name, float(worst.max()), int((~(worst <= 1.0)).sum()), worst.numel())


def check_lse_norms(got, want):
    value, bound = want
    empty = torch.isinf(value)
    assert torch.equal(torch.isinf(got), empty) and bool((got[empty] < 0).all())
    error = (got.to(F64) - value)[~empty].abs()
    assert bool((error <= bound[~empty]).all()), float((error / bound[~empty]).max())
