"""Cases and plain forms of the block operators: residual + RMS norm (BF16 or MXFP8 out), rotary positions, and
attention with a sliding window and visible first tokens.

`run(state)` makes one pass: with `own` the framework's operators (fuse_b200.block), without it the same formulas in
elementary torch operations, in 32 bits (angles in 64), rounded once at the end.  `exact` is the definition in 64 bits."""
import math

import torch

own = False

BF16 = torch.bfloat16
DEVICE = "cuda"

# Sizes follow the benchmark configurations of the projections: hidden 4096 / 5120 / 8192, heads of 128 with 8 KV heads,
# and what one rank of a context-parallel group holds between the two all-to-alls (a few heads, every position).
LISTED = [
    # one token's norm while answering: the launch is all there is
    dict(name="norm_one_row", op="norm", rows=1, hidden=5120, mxfp8=False, train=False),
    # what feeds the MXFP8 QKV projection: the rank's 16K tokens, residual added, bytes and scales out
    dict(name="norm_mxfp8_16k", op="norm", rows=16384, hidden=4096, mxfp8=True, train=False),
    # a training step's norm with both gradients, a row count that fills no tile
    dict(name="norm_train_odd", op="norm", rows=8191, hidden=8192, mxfp8=False, train=True),
    # one token's rotation while answering
    dict(name="rotary_one_row", op="rotary", rows=1, seq=1, start=70000, q_heads=32, kv_heads=8, head_dim=128,
         rotary_dim=128, interleaved=False, scaling="wavelength", given=False, train=False),
    # 128K positions of one rank's heads after the all-to-all, frequencies scaled for the long context
    dict(name="rotary_128k", op="rotary", rows=131072, seq=131072, start=0, q_heads=4, kv_heads=1, head_dim=128,
         rotary_dim=128, interleaved=False, scaling="wavelength", given=False, train=False),
    # a training step: half of each head rotated, interleaved pairs, positions from a tensor, ragged row count
    dict(name="rotary_train_part", op="rotary", rows=8209, seq=8209, start=0, q_heads=16, kv_heads=4, head_dim=128,
         rotary_dim=64, interleaved=True, scaling="yarn", given=True, train=True),
    # the shortest answer step: one token against a short context
    dict(name="attn_one_token", op="attention", batch=1, q_len=1, kv_len=257, q_heads=4, kv_heads=1, head_dim=64,
         window=0, sinks=0, ragged=False, train=False),
    # a batch of answer steps against long contexts: one token each, 16K keys
    dict(name="attn_few_rows_16k", op="attention", batch=8, q_len=1, kv_len=16384, q_heads=32, kv_heads=8, head_dim=128,
         window=0, sinks=0, ragged=False, train=False),
    # a prompt at context parallelism 8 of a 64 / 8 head model: 8 query heads on one KV head
    dict(name="attn_causal_8k", op="attention", batch=1, q_len=8192, kv_len=8192, q_heads=8, kv_heads=1, head_dim=128,
         window=0, sinks=0, ragged=False, train=False),
    # a long prompt with a sliding window and four sinks
    dict(name="attn_window_16k", op="attention", batch=1, q_len=16384, kv_len=16384, q_heads=4, kv_heads=1, head_dim=128,
         window=2048, sinks=4, ragged=False, train=False),
    # a training step, full causal
    dict(name="attn_train_8k", op="attention", batch=1, q_len=8192, kv_len=8192, q_heads=8, kv_heads=2, head_dim=128,
         window=0, sinks=0, ragged=False, train=True),
    # a training step on a padded batch of unequal lengths: heads of 64 in groups of three, window and sinks
    dict(name="attn_train_ragged", op="attention", batch=3, q_len=1537, kv_len=1537, q_heads=12, kv_heads=4, head_dim=64,
         window=256, sinks=3, ragged=True, train=True),
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "rotary", "attention"))
    if op == "norm":
        hidden = 32 * _log(rng, 4, 512)
        rows = _log(rng, 1, max(1, 16384 * 4096 // hidden))
        train = rng.random() < 0.5
        return dict(op=op, rows=rows, hidden=hidden, mxfp8=not train and rng.random() < 0.6, train=train)
    if op == "rotary":
        head_dim = rng.choice((64, 96, 128, 256))
        kv_heads = rng.choice((1, 2, 4, 8))
        q_heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
        rows = _log(rng, 1, 131072 * 640 // (head_dim * (q_heads + kv_heads)))
        return dict(op=op, rows=rows, seq=rng.choice((rows, max(1, rows // 3))), start=rng.choice((0, _log(rng, 1, 400000))),
                    q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice((head_dim, head_dim // 2, head_dim // 4)), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(("none", "linear", "ntk", "wavelength", "yarn")), given=rng.random() < 0.5,
                    train=rng.random() < 0.4)
    head_dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4))
    q_heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
    window = rng.choice((0, 0, _log(rng, 16, 4096)))
    sinks = rng.choice((0, _log(rng, 1, 300))) if window else 0
    shape = rng.random()
    if shape < 0.3:  # a few new tokens against what went before
        batch, q_len, train = _log(rng, 1, 8), _log(rng, 1, 16), False
        kv_len = q_len + _log(rng, 1, 16384)
    else:
        train = rng.random() < 0.5
        q_len = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(8, 4096 // q_len)))
        kv_len = q_len if rng.random() < 0.7 else q_len + _log(rng, 1, 2048)
    return dict(op=op, batch=batch, q_len=q_len, kv_len=kv_len, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                window=window, sinks=sinks, ragged=batch > 1 and rng.random() < 0.5, train=train)


# ------------------------------------------------------------------------------------------------ inputs
ROTARY = {"none": {}, "linear": dict(factor=4.0), "ntk": dict(factor=4.0),
          "wavelength": dict(factor=8.0, original_context=8192, low_freq_factor=1.0, high_freq_factor=4.0),
          "yarn": dict(factor=16.0, original_context=8192, beta_fast=32.0, beta_slow=1.0)}
THETA = 500000.0


def _randn(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE) * scale).to(BF16)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(1000003 * (seed % (1 << 31)) + 17)
    s = dict(case)
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        s["x"] = _randn(gen, rows, hidden)
        # a residual stream grows with depth and has a few large channels
        spread = torch.exp(torch.randn(hidden, generator=gen, device=DEVICE))
        s["residual"] = (torch.randn(rows, hidden, generator=gen, device=DEVICE) * spread).to(BF16)
        s["gamma"] = (1.0 + 0.2 * torch.randn(hidden, generator=gen, device=DEVICE)).to(BF16)
        if case["train"]:
            s["dy"], s["dh"] = _randn(gen, rows, hidden, scale=0.01), _randn(gen, rows, hidden, scale=0.01)
            for name in ("x", "residual", "gamma"):
                s[name].requires_grad_(own)
    elif case["op"] == "rotary":
        rows, d = case["rows"], case["head_dim"]
        s["q"], s["k"] = _randn(gen, rows, case["q_heads"] * d), _randn(gen, rows, case["kv_heads"] * d)
        s["positions"] = None
        if case["given"]:  # documents of unequal length in one row of tokens
            s["positions"] = case["start"] + torch.randint(0, max(1, case["seq"]), (rows,), generator=gen, device=DEVICE)
        if case["train"]:
            s["dq"], s["dk"] = _randn(gen, rows, case["q_heads"] * d, scale=0.01), _randn(gen, rows, case["kv_heads"] * d, scale=0.01)
            for name in ("q", "k"):
                s[name].requires_grad_(own)
    else:
        b, d = case["batch"], case["head_dim"]
        s["q"] = _randn(gen, b * case["q_len"], case["q_heads"] * d)
        s["k"] = _randn(gen, b * case["kv_len"], case["kv_heads"] * d)
        s["v"] = _randn(gen, b * case["kv_len"], case["kv_heads"] * d)
        s["q_lengths"] = s["kv_lengths"] = None
        if case["ragged"]:
            short = torch.randint(0, case["q_len"], (b,), generator=gen, device=DEVICE).to(torch.int32)
            short[0] = 0
            s["q_lengths"], s["kv_lengths"] = case["q_len"] - short, case["kv_len"] - short
        if case["train"]:
            s["do"] = _randn(gen, b * case["q_len"], case["q_heads"] * d)
            for name in ("q", "k", "v"):
                s[name].requires_grad_(own)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from fuse_b200 import block

    if s["op"] == "norm":
        if s["mxfp8"]:
            h, data, scales = block.rms_norm_mxfp8(s["x"], s["gamma"], residual=s["residual"])
            return {"h": h, "data": data.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}
        y, h = block.rms_norm(s["x"], s["gamma"], residual=s["residual"])
        if not s["train"]:
            return {"y": y, "h": h}
        dx, dgamma = torch.autograd.grad((y, h), (s["x"], s["gamma"]), (s["dy"], s["dh"]))
        return {"y": y, "h": h, "dx": dx, "dgamma": dgamma}
    if s["op"] == "rotary":
        spec = block.Rotary(rotary_dim=s["rotary_dim"], theta=THETA, interleaved=s["interleaved"], scaling=s["scaling"],
                            **ROTARY[s["scaling"]])
        q, k = block.rotary(s["q"], s["k"], spec, head_dim=s["head_dim"], seq_len=s["seq"], start=s["start"],
                            positions=s["positions"])
        if not s["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    o = block.attention(s["q"], s["k"], s["v"], batch=s["batch"], head_dim=s["head_dim"], causal=True, window=s["window"],
                        sinks=s["sinks"], q_lengths=s["q_lengths"], kv_lengths=s["kv_lengths"])
    if not s["train"]:
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_mxfp8(y):
    """E4M3 values and one power-of-two scale per 32 of a row, the scales in 512-byte atoms of 128 rows x 4 groups;
    2^0 where an atom reaches past the operand."""
    rows, k = y.shape
    groups = y.float().view(rows, k // 32, 32)
    mantissa, exponent = torch.frexp(groups.abs().amax(dim=2))
    # the smallest power of two that keeps the largest value within 448 = 1.75 * 2^8; 2^0 for a group of zeros
    exponent = torch.where(mantissa == 0, torch.zeros_like(exponent), exponent - 9 + (mantissa > 0.875).int())
    scale = torch.exp2(exponent.float())
    data = (groups / scale[:, :, None]).to(torch.float8_e4m3fn).view(rows, k)
    padded = torch.ones(-(-rows // 128) * 128, -(-k // 128) * 4, device=y.device)
    padded[:rows, :k // 32] = scale
    atoms = padded.view(-1, 4, 32, padded.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    return data, atoms.to(torch.float8_e8m0fnu)


def _plain_norm(s):
    h = (s["x"].float() + s["residual"].float()).to(BF16)
    hf, g = h.float(), s["gamma"].float()
    r = torch.rsqrt(hf.square().mean(dim=1, keepdim=True) + 1e-6)
    y = (hf * r * g).to(BF16)
    if s["mxfp8"]:
        data, scales = _plain_mxfp8(y)
        return {"h": h, "data": data, "scales": scales}
    if not s["train"]:
        return {"y": y, "h": h}
    dyf = s["dy"].float()
    n = hf * r
    dn = dyf * g
    dx = s["dh"].float() + r * (dn - n * (dn * n).mean(dim=1, keepdim=True))
    return {"y": y, "h": h, "dx": dx.to(BF16), "dgamma": (dyf * n).sum(dim=0).to(BF16)}


def _frequencies(rd, scaling, theta=THETA):
    """Radians per position of every pair, in 64 bits, and the factor on both outputs."""
    p = ROTARY[scaling]
    i = torch.arange(rd // 2, dtype=torch.float64, device=DEVICE)
    if scaling == "ntk":
        theta = theta * p["factor"] ** (rd / (rd - 2))
    f = theta ** (-2.0 * i / rd)
    if scaling == "linear":
        f = f / p["factor"]
    elif scaling == "wavelength":
        turns = p["original_context"] * f / (2.0 * math.pi)  # of the pair within the original context
        smooth = ((turns - p["low_freq_factor"]) / (p["high_freq_factor"] - p["low_freq_factor"])).clamp(0.0, 1.0)
        f = (1.0 - smooth) * f / p["factor"] + smooth * f
    elif scaling == "yarn":
        def pair(turns):
            return rd * math.log(p["original_context"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))
        low, high = max(math.floor(pair(p["beta_fast"])), 0), min(math.ceil(pair(p["beta_slow"])), rd - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - ramp) + f / p["factor"] * ramp
        return f, 0.1 * math.log(p["factor"]) + 1.0
    return f, 1.0


def _angles(s):
    positions = s["positions"]
    if positions is None:
        positions = s["start"] + torch.arange(s["rows"], device=DEVICE) % s["seq"]
    f, m = _frequencies(s["rotary_dim"], s["scaling"])
    a = positions.double()[:, None] * f
    return torch.cos(a) * m, torch.sin(a) * m


def _rotate(x, cos, sin, d, rd, interleaved):
    rows = x.shape[0]
    x = x.view(rows, -1, d)
    rot, rest = x[..., :rd], x[..., rd:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :rd // 2], rot[..., rd // 2:])
    c, t = cos[:, None, :], sin[:, None, :]
    u, v = a * c - b * t, a * t + b * c
    out = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((out, rest), dim=-1).view(rows, -1)


def _plain_rotary(s):
    cos, sin = (t.float() for t in _angles(s))
    layout = (s["head_dim"], s["rotary_dim"], s["interleaved"])
    out = {n: _rotate(s[n].float(), cos, sin, *layout).to(BF16) for n in ("q", "k")}
    if s["train"]:
        out.update({n: _rotate(s[n].float(), cos, -sin, *layout).to(BF16) for n in ("dq", "dk")})
    return out


def _visible(s, q_len, kv_len):
    """[batch, q_len, kv_len]: the query at position p = i + kv_length - q_length sees keys j <= p that lie within the
    window behind it or among the first `sinks`; nothing behind a sequence's length is seen or sees."""
    i, j = torch.arange(q_len, device=DEVICE)[None, :, None], torch.arange(kv_len, device=DEVICE)[None, None, :]
    ql = s["q_lengths"][:, None, None] if s["q_lengths"] is not None else q_len
    kl = s["kv_lengths"][:, None, None] if s["kv_lengths"] is not None else kv_len
    p = i + (kl - ql)
    seen = j <= p
    if s["window"]:
        seen = seen & ((p - j < s["window"]) | (j < s["sinks"]))
    return seen & (i < ql) & (j < kl)


def _heads(x, batch, length, heads, d):
    return x.view(batch, length, heads, d).transpose(1, 2)


def _plain_attention(s):
    b, ql, kl, hq, hk, d = (s[n] for n in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "head_dim"))
    g, scale = hq // hk, 1.0 / math.sqrt(d)
    q = _heads(s["q"].float(), b, ql, hq, d).reshape(b, hk, g, ql, d)
    k, v = (_heads(s[n].float(), b, kl, hk, d)[:, :, None] for n in ("k", "v"))
    seen = _visible(s, ql, kl)[:, None, None]
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp_min(-3.0e38)
    p = scores.sub_(top).exp_()
    p.div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-38))
    o = torch.matmul(p, v)

    def rows(x):
        return x.reshape(b, -1, x.shape[-2], d).transpose(1, 2).reshape(b * x.shape[-2], -1).to(BF16)

    if not s["train"]:
        return {"o": rows(o)}
    do = _heads(s["do"].float(), b, ql, hq, d).reshape(b, hk, g, ql, d)
    if s["q_lengths"] is not None:  # rows behind a sequence take no part
        do = do * (torch.arange(ql, device=DEVICE) < s["q_lengths"][:, None])[:, None, None, :, None]
    dv = torch.matmul(p.transpose(-1, -2), do).sum(dim=2)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = dp.sub_((do * o).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(dim=2)
    return {"o": rows(o), "dq": rows(dq), "dk": rows(dk), "dv": rows(dv)}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ work
def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, at full lengths."""
    ql, kl, w, n = case["q_len"], case["kv_len"], case["window"], case["sinks"]
    total = 0
    for i in range(ql):
        p = i + kl - ql
        total += p + 1 if not w else min(p + 1, w) + min(n, max(0, p + 1 - w))
    return total * case["batch"]


def work(case):
    if case["op"] == "norm":
        n, k = case["rows"] * case["hidden"], case["hidden"]
        if case["train"]:  # forward: x, residual in, y, h out; backward: dy, dh, h in, dx out
            return {"bytes": 16 * n + 4 * k, "flops": 15 * n}
        return {"bytes": 6 * n + (n + n / 32 if case["mxfp8"] else 2 * n) + 2 * k, "flops": 6 * n}
    if case["op"] == "rotary":
        n = case["rows"] * (case["q_heads"] + case["kv_heads"]) * case["head_dim"]
        times = 2 if case["train"] else 1
        return {"bytes": times * (4 * n + (8 * case["rows"] if case["given"] else 0)), "flops": times * 3 * n}
    d = case["head_dim"]
    q, kv = (case["batch"] * case[a] * case[h] * d for a, h in (("q_len", "q_heads"), ("kv_len", "kv_heads")))
    pairs = _pairs(case) * case["q_heads"]
    if case["train"]:  # two products forward, five backward
        return {"bytes": 2 * (4 * q + 4 * kv) + 2 * q, "flops": 14 * d * pairs}
    return {"bytes": 2 * (2 * q + 2 * kv), "flops": 4 * d * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    if case["op"] == "norm":
        # the stream is a BF16 tensor by definition, and the norm is that of the stream
        h = (s["x"].double() + s["residual"].double()).to(BF16).double()
        g = s["gamma"].double()
        rms = torch.sqrt((h * h).sum(1, keepdim=True) / case["hidden"] + 1e-6)
        y = h / rms * g
        if case["mxfp8"]:
            # the bytes are those of the BF16 output; 2^e >= amax / 448 is the smallest such power
            yb = y.to(BF16).double()
            blocks = yb.reshape(case["rows"], -1, 32)
            top = blocks.abs().amax(2)
            e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0))
            scale = torch.where(top > 0, torch.exp2(e), torch.ones_like(e))
            ratio = blocks / scale[..., None]
            step = torch.exp2(torch.floor(torch.log2(ratio.abs().clamp_min(2.0 ** -6))) - 3.0)
            data = (torch.round(ratio / step) * step).reshape(yb.shape)  # round to nearest even
            tiles_m, tiles_k = -(-case["rows"] // 128), -(-case["hidden"] // 128)
            grid = torch.ones(tiles_m * 128, tiles_k * 4, dtype=torch.float64, device=DEVICE)
            grid[:case["rows"], :scale.shape[1]] = scale
            out = torch.empty(tiles_m, tiles_k, 32, 4, 4, dtype=torch.float64, device=DEVICE)
            for quarter in range(4):
                out[:, :, :, quarter] = grid.view(tiles_m, 4, 32, tiles_k, 4)[:, quarter].transpose(1, 2)
            return {"h": h, "data": data, "scales": out.reshape(-1)}
        if not case["train"]:
            return {"y": y, "h": h}
        dy, dh = s["dy"].double(), s["dh"].double()
        w = dy * g
        dx = dh + w / rms - h * (w * h).sum(1, keepdim=True) / (case["hidden"] * rms ** 3)
        return {"y": y, "h": h, "dx": dx, "dgamma": (dy * h / rms).sum(0)}
    if case["op"] == "rotary":
        cos, sin = _angles(s)
        turn = torch.complex(cos, sin)[:, None, :]
        d, rd = case["head_dim"], case["rotary_dim"]

        def turned(x, by):
            x = x.double().reshape(case["rows"], -1, d)
            out = x.clone()
            if case["interleaved"]:
                z = torch.view_as_complex(x[..., :rd].reshape(*x.shape[:2], rd // 2, 2).contiguous()) * by
                out[..., 0:rd:2], out[..., 1:rd:2] = z.real, z.imag
            else:
                z = torch.complex(x[..., :rd // 2].contiguous(), x[..., rd // 2:rd].contiguous()) * by
                out[..., :rd // 2], out[..., rd // 2:rd] = z.real, z.imag
            return out.reshape(case["rows"], -1)

        out = {n: turned(s[n], turn) for n in ("q", "k")}
        if case["train"]:
            out.update({n: turned(s[n], turn.conj()) for n in ("dq", "dk")})
        return out
    b, ql, kl, hq, hk, d = (case[n] for n in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "head_dim"))
    out = {"o": torch.zeros(b * ql, hq * d, dtype=torch.float64, device=DEVICE)}
    if case["train"]:
        out.update(dq=torch.zeros_like(out["o"]), dk=torch.zeros(b * kl, hk * d, dtype=torch.float64, device=DEVICE),
                   dv=torch.zeros(b * kl, hk * d, dtype=torch.float64, device=DEVICE))
    ones = torch.ones(b, dtype=torch.int64)
    qls = s["q_lengths"].tolist() if s["q_lengths"] is not None else (ones * ql).tolist()
    kls = s["kv_lengths"].tolist() if s["kv_lengths"] is not None else (ones * kl).tolist()
    for n in range(b):
        nq, nk = qls[n], kls[n]
        pos = torch.arange(nk - nq, nk, device=DEVICE)[:, None]
        key = torch.arange(nk, device=DEVICE)[None, :]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | ((key <= pos - case["window"]) & (key >= case["sinks"]))
        empty = hidden.all(dim=1, keepdim=True)
        for h in range(hq):
            kv = h // (hq // hk)
            rq, cq = slice(n * ql, n * ql + nq), slice(h * d, h * d + d)
            rk, ck = slice(n * kl, n * kl + nk), slice(kv * d, kv * d + d)
            q, k, v = s["q"][rq, cq].double(), s["k"][rk, ck].double(), s["v"][rk, ck].double()
            w = torch.softmax((q @ k.T / d ** 0.5).masked_fill(hidden, -math.inf), dim=1)
            w = torch.where(empty, torch.zeros_like(w), w)
            out["o"][rq, cq] = w @ v
            if case["train"]:
                do = s["do"][rq, cq].double()
                dw = do @ v.T
                ds = w * (dw - (w * dw).sum(1, keepdim=True)) / d ** 0.5
                out["dq"][rq, cq] = ds @ k
                out["dk"][rk, ck] += ds.T @ q
                out["dv"][rk, ck] += w.T @ do
    return out
