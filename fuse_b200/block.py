"""The operators of a transformer block between and before the fused projections, on torch tensors.

    y, h = rms_norm(x, gamma, residual=h)                 # -> proj.qkv(y, w_qkv)
    h, data, scales = rms_norm_mxfp8(x, gamma, h)         # -> the MXFP8 QKV projection's prequantised activation
    q, k = rotary(q, k, Rotary(128), head_dim=128)        # on the planar Q and K the all-to-all leaves

Tensors are BF16 [rows, width] on one CUDA device, rows `width` apart or more (views of wider tensors
do, with row strides of a multiple of 8 elements); a tensor that an operator cannot take is refused, never copied.
Work runs on the tensors' device and on its current stream.  Gradients come through torch.autograd
where an argument requires them; forward mode is refused.  The C entry points underneath are in include/fuse_b200.h."""
from __future__ import annotations

import ctypes as C
import dataclasses

import torch
from torch.autograd import forward_ad

from . import _native as N

BF16 = torch.bfloat16


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} -> cudaError {rc}")


def _refused(rc: int, what: str, tensors: dict, **limits: bool) -> None:
    """Raises for a launch that gave `rc`, with what of its arguments explains it: rows that are not where vectors can be
    read, and the limits that are not kept (description=whether it is)."""
    reasons = [f"{name} is not on a 16-byte boundary" for name, t in tensors.items() if t is not None and t.numel() and t.data_ptr() % 16]
    reasons += [f"{name}'s rows are {t.stride(0)} elements apart, not a multiple of 8 from {t.shape[1]} on"
                for name, t in tensors.items()
                if t is not None and t.dim() == 2 and t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < t.shape[1])]
    reasons += [name for name, kept in limits.items() if not kept]
    raise RuntimeError(f"{what} -> cudaError {rc}" + (": " + "; ".join(reasons) if reasons else ""))


def _within(bits: int, **numbers: int) -> None:
    """Whole numbers that a record's signed field of `bits` holds (ctypes would cut off the rest without a word).
    Names what does not; callers look first whether anything is that large, as the loop is a microsecond of a call's twenty."""
    for name, value in numbers.items():
        if not -(1 << (bits - 1)) <= value < 1 << (bits - 1):
            raise ValueError(f"{name}: {value} does not fit {bits} bits")


def _rows(t: torch.Tensor, name: str, width: int | None = None, rows: int | None = None, device=None) -> None:
    if (not isinstance(t, torch.Tensor) or t.dtype != BF16 or t.dim() != 2 or not t.is_cuda or
            (t.shape[1] != 1 and t.stride(1) != 1) or (width is not None and t.shape[1] != width) or
            (rows is not None and t.shape[0] != rows) or (device is not None and t.device != device)):
        raise ValueError(f"{name}: expected a bfloat16 CUDA tensor [{'rows' if rows is None else rows}, "
                         f"{'width' if width is None else width}] with contiguous rows"
                         f"{'' if device is None else f' on {device}'}, got "
                         f"{(t.dtype, tuple(t.shape), t.stride(), t.device) if isinstance(t, torch.Tensor) else type(t)}")


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else -1


def _grad(g: torch.Tensor) -> torch.Tensor:
    """A gradient as autograd hands it over (it may be expanded, transposed or unaligned) as rows an operator takes."""
    if g.stride(1) == 1 and g.data_ptr() % 16 == 0 and (g.shape[0] == 1 or (g.stride(0) >= g.shape[1] and g.stride(0) % 8 == 0)):
        return g
    return g.clone(memory_format=torch.contiguous_format)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the rows of two tensors reach a common element (columns of one wider tensor, side by side, do not)."""
    if not a.numel() or not b.numel():
        return False
    if a.data_ptr() > b.data_ptr():
        a, b = b, a
    gap, (n, width), (m, other) = (b.data_ptr() - a.data_ptr()) // a.element_size(), a.shape, b.shape
    if gap >= (n - 1) * a.stride(0) + width:
        return False
    pitch = a.stride(0)
    if n == 1 or pitch < width:
        return True
    # b's rows against a's: with one pitch all of them start in the same column, and the first decides
    for at in range(gap, gap + 1 if m == 1 or b.stride(0) == pitch else gap + m * b.stride(0), max(b.stride(0), 1)):
        row, column = divmod(at, pitch)
        if (row < n and column < width) or (row + 1 < n and column + other > pitch):
            return True
    return False


try:  # the stream's handle without the Stream object around it: 0.1 us instead of 1.4
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


class _On:
    """Makes a tensor's device the current one for a launch, where it is not already, and hands out its stream."""
    __slots__ = ("index", "back")

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index

    def __enter__(self):
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _written(*tensors) -> None:
    """What a kernel has written through its pointer counts as modified in place: autograd then refuses a backward that had
    saved it, as it does for torch's own in-place operations."""
    for t in tensors:
        if t is not None:
            torch.autograd.graph.increment_version(t)


def _wants_grad(*tensors) -> bool:
    # a tensor in forward mode need not require a gradient; its tangent would be dropped, that is, taken for zero
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the block operators have no forward-mode derivative (torch.autograd.forward_ad, torch.func.jvp)")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------ RMS norm
def _norm_arguments(x, gamma, residual):
    _rows(x, "x")
    if residual is not None:
        _rows(residual, "residual", x.shape[1], x.shape[0], x.device)
    if gamma.dtype != BF16 or tuple(gamma.shape) != (x.shape[1],) or not gamma.is_contiguous() or gamma.device != x.device:
        raise ValueError(f"gamma: expected contiguous bfloat16 ({x.shape[1]},) on {x.device}, got {gamma.dtype} "
                         f"{tuple(gamma.shape)} on {gamma.device}")


def _norm_forward(x, gamma, residual, eps, output: bool, mxfp8: bool):
    rows, hidden = x.shape
    p = N.RmsNormParams()
    p.input, p.gamma, p.rows, p.hidden, p.epsilon = x.data_ptr(), gamma.data_ptr(), rows, hidden, eps
    p.input_stride = _stride(x)
    p.residual_output_stride = p.output_stride = -1
    h, y, data, scales = x, None, None, None
    if residual is not None:
        h = torch.empty((rows, hidden), dtype=BF16, device=x.device)
        p.residual, p.residual_stride, p.residual_output = residual.data_ptr(), _stride(residual), h.data_ptr()
    if output:
        y = torch.empty((rows, hidden), dtype=BF16, device=x.device)
        p.output = y.data_ptr()
    if mxfp8:
        if hidden % 32:
            raise ValueError(f"an MXFP8 output needs rows of a multiple of 32 elements, got {hidden}")
        data = torch.empty((rows, hidden), dtype=torch.uint8, device=x.device)
        scales = torch.empty(N.lib().fuse_b200_mxfp8_scale_bytes(rows, hidden), dtype=torch.uint8, device=x.device)
        p.quantized.data, p.quantized.scales = data.data_ptr(), scales.data_ptr()
        p.quantized.data_bytes, p.quantized.scale_bytes = data.numel(), scales.numel()
    if rows:
        with _On(x) as stream:
            rc = N.lib().fuse_b200_launch_rms_norm(C.byref(p), stream)
        if rc:
            _refused(rc, "launch_rms_norm", dict(x=x, gamma=gamma, residual=residual), **{
                "hidden is a multiple of 8, at most 16384": hidden % 8 == 0 and hidden <= 16384, "eps is at least 1e-30": eps >= 1e-30})
    return y, h, data, scales


def _norm_backward(dy, dh, h, gamma, eps, want_gamma: bool):
    rows, hidden = h.shape
    p = N.RmsNormBackwardParams()
    dy = _grad(dy)
    dx = torch.empty((rows, hidden), dtype=BF16, device=h.device)
    p.grad_output, p.grad_output_stride = dy.data_ptr(), _stride(dy)
    p.stream_input, p.stream_input_stride = h.data_ptr(), _stride(h)
    if dh is not None:
        dh = _grad(dh)
        p.grad_stream, p.grad_stream_stride = dh.data_ptr(), _stride(dh)
    p.gamma, p.grad_input, p.grad_input_stride = gamma.data_ptr(), dx.data_ptr(), -1
    p.rows, p.hidden, p.epsilon = rows, hidden, eps
    dgamma = None
    with _On(h) as stream:
        if want_gamma:
            size = C.c_size_t()
            _check(N.lib().fuse_b200_rms_norm_backward_workspace_size(rows, hidden, C.byref(size)),
                   "rms_norm_backward_workspace_size")
            workspace = torch.empty(size.value, dtype=torch.uint8, device=h.device)
            dgamma = torch.empty(hidden, dtype=BF16, device=h.device)
            p.grad_gamma, p.workspace, p.workspace_bytes = dgamma.data_ptr(), workspace.data_ptr(), size.value
        _check(N.lib().fuse_b200_launch_rms_norm_backward(C.byref(p), stream), "launch_rms_norm_backward")
    return dx, dgamma


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, residual, eps, mxfp8):
        y, h, data, scales = _norm_forward(x, gamma, residual, eps, True, mxfp8)
        ctx.save_for_backward(h, gamma)
        ctx.eps, ctx.summed = eps, residual is not None
        ctx.set_materialize_grads(False)
        if mxfp8:
            ctx.mark_non_differentiable(data, scales)
        return y, h if residual is not None else None, data, scales

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh, _data, _scales):
        h, gamma = ctx.saved_tensors
        if dy is None:
            return dh, None, dh if ctx.summed else None, None, None
        dx, dgamma = _norm_backward(dy, dh, h, gamma, ctx.eps, ctx.needs_input_grad[1])
        return dx, dgamma, dx if ctx.summed else None, None, None


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6,
             mxfp8: bool = False):
    """h = x + residual (BF16, or x itself without a residual); y = h / sqrt(mean(h^2) + eps) * gamma.
    Returns (y, h), with `mxfp8` (y, h, data, scales): the E4M3 bytes [rows, hidden] of y and its UE8M0 scales in
    native atoms, what the MXFP8 projections take.  hidden: a multiple of 8 (32 with mxfp8), at most 16384."""
    _norm_arguments(x, gamma, residual)
    if _wants_grad(x, gamma, residual):
        y, h, data, scales = _RmsNorm.apply(x, gamma, residual, eps, mxfp8)
        h = x if residual is None else h
    else:
        y, h, data, scales = _norm_forward(x, gamma, residual, eps, True, mxfp8)
    return (y, h, data, scales) if mxfp8 else (y, h)


def rms_norm_mxfp8(x: torch.Tensor, gamma: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """The same with the MXFP8 form alone, for a forward pass that keeps no BF16 activation: (h, data, scales).
    It has no gradient; a training step takes rms_norm(..., mxfp8=True)."""
    _norm_arguments(x, gamma, residual)
    if _wants_grad(x, gamma, residual):
        raise RuntimeError("rms_norm_mxfp8 has no gradient: use rms_norm(..., mxfp8=True), or torch.no_grad()")
    _, h, data, scales = _norm_forward(x, gamma, residual, eps, False, True)
    return h, data, scales


# ------------------------------------------------------------------------------------------------ rotary positions
@dataclasses.dataclass(frozen=True)
class Rotary:
    """What turns: the first `rotary_dim` elements of every head, pairs (i, i + rotary_dim / 2) or, interleaved,
    (2i, 2i + 1), at theta^(-2i / rotary_dim) radians per position, scaled for contexts longer than
    `original_context` by "linear", "ntk", "wavelength" or "yarn" (include/fuse_b200.h has the formulas).
    `magnitude` multiplies cosine and sine (default: 1, or yarn's 0.1 ln(factor) + 1)."""
    rotary_dim: int
    theta: float = 10000.0
    interleaved: bool = False
    scaling: str = "none"
    factor: float = 1.0
    original_context: int = 0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    magnitude: float = 0.0

    def record(self) -> N.RotarySpec:
        if self.scaling not in N.ROTARY_SCALINGS:
            raise ValueError(f"scaling: one of {sorted(N.ROTARY_SCALINGS)}, got {self.scaling!r}")
        if abs(self.rotary_dim) >= 1 << 31 or abs(self.original_context) >= 1 << 63:
            _within(32, rotary_dim=self.rotary_dim)
            _within(64, original_context=self.original_context)
        return N.RotarySpec(self.theta, self.factor, self.low_freq_factor, self.high_freq_factor, self.beta_fast,
                            self.beta_slow, self.magnitude, self.original_context, self.rotary_dim,
                            N.ROTARY_SCALINGS[self.scaling], 1 if self.interleaved else 0)

    def frequencies(self) -> tuple[list[float], float]:
        """Radians per position of every pair, and the magnitude."""
        from . import api
        rc, values, magnitude = api.rotary_frequencies(self.record())
        if rc != 0:
            raise ValueError(f"not a rotary specification: {self}")
        return values, magnitude


def _rotary_launch(q, k, qo, ko, spec, head_dim, seq_len, start, positions, adjoint):
    p = N.RotaryParams()
    if q is not None:
        p.q, p.q_output, p.q_heads = q.data_ptr(), qo.data_ptr(), q.shape[1] // head_dim
        p.q_stride, p.q_output_stride = _stride(q), _stride(qo)
    if k is not None:
        p.k, p.k_output, p.kv_heads = k.data_ptr(), ko.data_ptr(), k.shape[1] // head_dim
        p.k_stride, p.k_output_stride = _stride(k), _stride(ko)
    if positions is not None:
        p.positions, p.position_bytes = positions.data_ptr(), positions.element_size()
    some = q if q is not None else k
    p.position_start, p.rows, p.seq_len = start, some.shape[0], seq_len
    p.head_dim, p.spec, p.adjoint = head_dim, spec, adjoint
    with _On(some) as stream:
        rc = N.lib().fuse_b200_launch_rotary(C.byref(p), stream)
    if rc:
        raise RuntimeError(f"launch_rotary -> cudaError {rc}" + (
            f": rotary_dim is even and within 2 .. head_dim, at most 256, got {spec.rotary_dim} of {head_dim}"
            if not 2 <= spec.rotary_dim <= min(head_dim, 256) or spec.rotary_dim % 2 else
            ": the specification's scaling has no such parameters" if N.lib().fuse_b200_rotary_frequencies(
                C.byref(spec), (C.c_double * 128)(), C.byref(C.c_double())) else ""))


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, spec, head_dim, seq_len, start, positions):
        ctx.rest = (spec, head_dim, seq_len, start)
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        qo, ko = (None if t is None else torch.empty(t.shape, dtype=BF16, device=t.device) for t in (q, k))
        _rotary_launch(q, k, qo, ko, spec, head_dim, seq_len, start, positions, 0)
        return qo, ko

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, = ctx.saved_tensors
        dq, dk = (_grad(g) if g is not None and needed else None for g, needed in zip((dq, dk), ctx.needs_input_grad))
        if dq is None and dk is None:
            return (None,) * 7
        oq, ok = (None if g is None else torch.empty(g.shape, dtype=BF16, device=g.device) for g in (dq, dk))
        spec, head_dim, seq_len, start = ctx.rest
        _rotary_launch(dq, dk, oq, ok, spec, head_dim, seq_len, start, positions, 1)
        return oq, ok, None, None, None, None, None


def _rotary_arguments(q, k, spec, head_dim, seq_len, start, positions):
    some = q if q is not None else k
    if some is None:
        raise ValueError("rotary needs q or k")
    for t, name in ((q, "q"), (k, "k")):
        if t is not None:
            _rows(t, name, rows=some.shape[0], device=some.device)
            if head_dim <= 0 or t.shape[1] % head_dim:
                raise ValueError(f"{name}: rows of {t.shape[1]} elements are not whole heads of {head_dim}")
    if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous() or
                                  tuple(positions.shape) != (some.shape[0],) or positions.device != some.device):
        raise ValueError(f"positions: expected contiguous int32 or int64 ({some.shape[0]},) on {some.device}")
    if seq_len is None:
        seq_len = max(1, some.shape[0])
    if abs(seq_len) >= 1 << 63 or abs(start) >= 1 << 63:
        _within(64, seq_len=seq_len, start=start)
    return spec.record(), seq_len


def rotary(q: torch.Tensor | None, k: torch.Tensor | None, spec: Rotary, *, head_dim: int, seq_len: int | None = None,
           start: int = 0, positions: torch.Tensor | None = None):
    """Turned copies of q [rows, q_heads * head_dim] and k [rows, kv_heads * head_dim] (either may be None).  Row r is
    at position positions[r], or start + r % seq_len (seq_len: all rows, one sequence)."""
    record, seq_len = _rotary_arguments(q, k, spec, head_dim, seq_len, start, positions)
    if _wants_grad(q, k):
        return _Rotary.apply(q, k, record, head_dim, seq_len, start, positions)
    qo, ko = (None if t is None else torch.empty(t.shape, dtype=BF16, device=t.device) for t in (q, k))
    _rotary_launch(q, k, qo, ko, record, head_dim, seq_len, start, positions, 0)
    return qo, ko


def rotary_(q: torch.Tensor | None, k: torch.Tensor | None, spec: Rotary, *, head_dim: int, seq_len: int | None = None,
            start: int = 0, positions: torch.Tensor | None = None):
    """The same in place (no gradient); q and k must not share memory."""
    record, seq_len = _rotary_arguments(q, k, spec, head_dim, seq_len, start, positions)
    if _wants_grad(q, k):
        raise RuntimeError("rotary_ writes its arguments and has no gradient: use rotary")
    if q is not None and k is not None and _overlap(q, k):
        raise ValueError("q and k share memory: each would be turned while the other is read")
    _rotary_launch(q, k, q, k, record, head_dim, seq_len, start, positions, 0)
    _written(q, k)
    return q, k


# ------------------------------------------------------------------------------------------------ attention
def _attention_record(q, k, v, shape):
    """The launch record without outputs; `shape`: the scalars every launch of this call shares."""
    batch, q_len, kv_len, q_heads, kv_heads, head_dim, causal, window, sinks, scale, q_starts, q_lengths, kv_starts, kv_lengths = shape
    p = N.AttentionParams()
    p.q, p.k, p.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    p.q_stride, p.k_stride, p.v_stride = _stride(q), _stride(k), _stride(v)
    p.q_rows, p.kv_rows = q.shape[0], k.shape[0]
    if q_starts is not None:
        p.q_starts = q_starts.data_ptr()
    if q_lengths is not None:
        p.q_lengths = q_lengths.data_ptr()
    if kv_starts is not None:
        p.kv_starts = kv_starts.data_ptr()
    if kv_lengths is not None:
        p.kv_lengths = kv_lengths.data_ptr()
    p.batch, p.q_len, p.kv_len = batch, q_len, kv_len
    p.q_heads, p.kv_heads, p.head_dim = q_heads, kv_heads, head_dim
    p.causal, p.window, p.sinks, p.scale = causal, window, sinks, scale
    return p


def _partial(q, k, shape) -> bool:
    """Whether some rows may belong to no sequence."""
    return any(t is not None for t in shape[10:]) or shape[0] * shape[1] != q.shape[0] or shape[0] * shape[2] != k.shape[0]


def _attention_forward(q, k, v, shape, out, want_lse, rest=None):
    ragged = _partial(q, k, shape)
    if out is None:  # rows of no sequence are zeros here; the operator leaves them as they are
        out = (torch.zeros if ragged else torch.empty)(q.shape, dtype=BF16, device=q.device)
    p = _attention_record(q, k, v, shape)
    p.output, p.output_stride = out.data_ptr(), _stride(out)
    if rest is not None:
        p.output_rest = rest.data_ptr()
    lse = None
    if want_lse:
        lse = torch.empty((shape[3], q.shape[0]), dtype=torch.float32, device=q.device)
        if ragged and want_lse == "whole":
            lse.fill_(-torch.inf)
        p.lse = lse.data_ptr()
    with _On(q) as stream:
        size = C.c_size_t()
        rc = N.lib().fuse_b200_attention_workspace_size(C.byref(p), C.byref(size))
        if not rc:
            if size.value:
                workspace = torch.empty(size.value, dtype=torch.uint8, device=q.device)
                p.workspace, p.workspace_bytes = workspace.data_ptr(), size.value
            rc = N.lib().fuse_b200_launch_attention(C.byref(p), None, stream)
    if rc:
        _refused(rc, "launch_attention", dict(q=q, k=k, v=v, out=out), **{
            "head_dim is 64 or 128": p.head_dim in (64, 128), "scale is positive and finite": 0.0 < p.scale < float("inf"),
            "q_len and kv_len are not negative": p.q_len >= 0 and p.kv_len >= 0,
            "batch * q_len rows are in q": shape[10] is not None or p.batch * p.q_len <= p.q_rows,
            "batch * kv_len rows are in k and v": shape[12] is not None or p.batch * p.kv_len <= p.kv_rows})
    return out, lse


def _attention_backward(do, q, k, v, out, rest, lse, shape):
    # one allocation (and, where rows may belong to no sequence, one clearing) for the three
    make = torch.zeros if _partial(q, k, shape) or not q.shape[0] else torch.empty
    nq, nk = q.shape[0] * q.shape[1], k.shape[0] * k.shape[1]
    gap = -nq % 8  # the parts start on 16-byte boundaries
    whole = make(nq + gap + 2 * nk, dtype=BF16, device=q.device)
    dq, dk, dv = whole[:nq].view(q.shape), whole[nq + gap:nq + gap + nk].view(k.shape), whole[nq + gap + nk:].view(v.shape)
    if not q.shape[0]:
        return dq, dk, dv
    do = _grad(do)
    p = N.AttentionBackwardParams()
    p.forward = _attention_record(q, k, v, shape)
    p.forward.output, p.forward.output_stride, p.forward.lse = out.data_ptr(), _stride(out), lse.data_ptr()
    p.forward.output_rest = rest.data_ptr()
    p.grad_output, p.grad_output_stride = do.data_ptr(), _stride(do)
    p.grad_q, p.grad_k, p.grad_v = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    p.grad_q_stride = p.grad_k_stride = p.grad_v_stride = -1
    with _On(q) as stream:
        size = C.c_size_t()
        _check(N.lib().fuse_b200_attention_backward_workspace_size(C.byref(p), C.byref(size)),
               "attention_backward_workspace_size")
        workspace = torch.empty(size.value, dtype=torch.uint8, device=q.device)
        p.workspace, p.workspace_bytes = workspace.data_ptr(), size.value
        _check(N.lib().fuse_b200_launch_attention_backward(C.byref(p), None, stream), "launch_attention_backward")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, shape, want_lse):
        # what rounding takes off the output, a byte an element: rowsum(do * out) would carry it into every gradient
        rest = torch.empty(q.shape, dtype=torch.int8, device=q.device)
        out, lse = _attention_forward(q, k, v, shape, None, want_lse, rest)
        ctx.save_for_backward(q, k, v, out, rest, lse, *shape[10:])
        ctx.shape = shape[:10]
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, _lse):
        q, k, v, out, rest, lse, *rows = ctx.saved_tensors
        dq, dk, dv = _attention_backward(do, q, k, v, out, rest, lse, (*ctx.shape, *rows))
        return dq, dk, dv, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, head_dim: int, batch: int = 1, causal: bool = True,
              window: int = 0, sinks: int = 0, scale: float | None = None, q_len: int | None = None,
              kv_len: int | None = None, q_starts: torch.Tensor | None = None, q_lengths: torch.Tensor | None = None,
              kv_starts: torch.Tensor | None = None, kv_lengths: torch.Tensor | None = None,
              out: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v per head: q [rows, q_heads * head_dim], k and v [kv_rows, kv_heads * head_dim] -> like q.

    The rows are `batch` sequences of q_len queries and kv_len keys (default: all rows, evenly), one behind the other.
    Shorter ones have their lengths in q_lengths / kv_lengths, others their first rows in q_starts / kv_starts
    (int32 [batch] on the device; q_len and kv_len are then the longest: what a length has beyond them is
    cut off).  Sequences may share keys (equal kv_starts) only without gradients, and never queries.  Queries are the last q_length positions of their sequence.  With `causal`,
    `window` limits a query to the last `window` keys up to its own and the first `sinks` of the sequence.  Rows of
    no sequence are zeros in the result (with `out`: as they were).
    `out`: a tensor to write to, such as UlyssesProjections.attention_buffer() -- without gradients only, since a
    later call would overwrite what the backward needs; it must not share memory with q, k or v.  `return_lse`: also FP32 [q_heads, rows], no gradient."""
    _rows(q, "q")
    _rows(k, "k", device=q.device)
    _rows(v, "v", k.shape[1], k.shape[0], q.device)
    if head_dim <= 0 or q.shape[1] % head_dim or k.shape[1] % head_dim or k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"heads of {head_dim}: rows of {q.shape[1]} (q) and {k.shape[1]} (k, v) elements are not whole groups")
    if batch <= 0 or (q_len is None and q.shape[0] % batch) or (kv_len is None and k.shape[0] % batch):
        raise ValueError(f"{q.shape[0]} queries and {k.shape[0]} keys are not {batch} sequences")
    for t, name in ((q_starts, "q_starts"), (q_lengths, "q_lengths"), (kv_starts, "kv_starts"), (kv_lengths, "kv_lengths")):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (batch,) or not t.is_contiguous() or t.device != q.device):
            raise ValueError(f"{name}: expected contiguous int32 ({batch},) on {q.device}")
    if window < 0 or sinks < 0 or (window and not causal):
        raise ValueError("window and sinks are not negative, and a window goes with causal attention")
    q_len, kv_len = q.shape[0] // batch if q_len is None else q_len, k.shape[0] // batch if kv_len is None else kv_len
    if max(batch, q_len, kv_len, window, sinks) >= 1 << 31 or min(q_len, kv_len) < 0:
        _within(32, batch=batch, q_len=q_len, kv_len=kv_len, window=window, sinks=sinks)
    shape = (batch, q_len, kv_len,
             q.shape[1] // head_dim, k.shape[1] // head_dim, head_dim, 1 if causal else 0, window, sinks,
             head_dim ** -0.5 if scale is None else scale, q_starts, q_lengths, kv_starts, kv_lengths)
    if out is not None:
        _rows(out, "out", q.shape[1], q.shape[0], q.device)
        if _wants_grad(out):
            raise RuntimeError("out= is written in place and must not require a gradient: pass out.detach(), or use torch.no_grad()")
        for t, name in ((q, "q"), (k, "k"), (v, "v")):
            if _overlap(out, t):
                raise ValueError(f"out and {name} share memory")
    if _wants_grad(q, k, v):
        if out is not None:
            raise RuntimeError("out= would be overwritten before the backward has read it: leave it out, or use torch.no_grad()")
        out, lse = _Attention.apply(q, k, v, shape, "whole" if return_lse else "own")
    else:
        given = out
        out, lse = _attention_forward(q, k, v, shape, given, "whole" if return_lse else None)
        _written(given)
    return (out, lse) if return_lse else out
