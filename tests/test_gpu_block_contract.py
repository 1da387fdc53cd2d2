"""What the block operators (fuse_b200/block.py) owe to autograd and to their arguments: writes that autograd sees, forward-mode
tangents, memory that two arguments share, numbers past 31 bits, the gradient of
the norm with two outputs."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from fuse_b200 import block

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
SPEC = block.Rotary(64)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(BF16)


# ---- writes in place are seen
def test_a_tensor_turned_in_place_is_not_taken_for_the_saved_one():
    q, k, v = (randn(40, 64, seed=i).requires_grad_() for i in range(3))
    kept = k * 1  # no leaf
    o = block.attention(q, kept, v, head_dim=64)
    with torch.no_grad():
        block.rotary_(None, kept, SPEC, head_dim=64)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_an_output_written_over_a_saved_tensor_is_not_taken_for_it():
    q, k, v = (randn(40, 64, seed=i).requires_grad_() for i in range(3))
    kept = q * 1
    o = block.attention(kept, k, v, head_dim=64)
    with torch.no_grad():
        block.attention(k, k, v, head_dim=64, out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_versions_count_writes():
    q, k = randn(8, 128), randn(8, 64)
    before = q._version, k._version
    block.rotary(q, k, SPEC, head_dim=64)
    assert (q._version, k._version) == before
    block.rotary_(q, k, SPEC, head_dim=64)
    assert q._version > before[0] and k._version > before[1]
    out = torch.empty_like(k)
    before = out._version
    block.attention(k, k, k, head_dim=64, out=out)
    assert out._version > before
    with torch.inference_mode():  # inference tensors have no versions
        block.rotary_(q.clone(), None, SPEC, head_dim=64)
        block.attention(k, k, k, head_dim=64, out=torch.empty_like(k))


# ---- forward mode has no derivative here: refused, not dropped
def test_forward_mode_is_refused():
    x, gamma, q, k, v = randn(8, 256), randn(256), randn(8, 64), randn(8, 64), randn(8, 64)
    calls = [(x, lambda t: block.rms_norm(t, gamma)), (gamma, lambda t: block.rms_norm(x, t)), (x, lambda t: block.rms_norm(x, gamma, t)),
             (x, lambda t: block.rms_norm(t, gamma, mxfp8=True)), (x, lambda t: block.rms_norm_mxfp8(t, gamma)),
             (q, lambda t: block.rotary(t, k, SPEC, head_dim=64)), (k, lambda t: block.rotary(q, t, SPEC, head_dim=64)),
             (q, lambda t: block.rotary_(t, None, SPEC, head_dim=64)),
             (q, lambda t: block.attention(t, k, v, head_dim=64)), (k, lambda t: block.attention(q, t, v, head_dim=64)),
             (v, lambda t: block.attention(q, k, t, head_dim=64))]
    for primal, call in calls:
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward"):
                call(forward_ad.make_dual(primal.clone(), torch.ones_like(primal)))
            call(primal.clone())  # without a tangent it runs
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (primal,), (torch.ones_like(primal),))


def test_an_output_of_its_own_derivative_is_refused():
    q, out = randn(8, 64), randn(8, 64, seed=1)
    keep = out.clone()
    with pytest.raises(RuntimeError, match="gradient"):
        block.attention(q, q, q, head_dim=64, out=out.requires_grad_())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward"):
        block.attention(q, q, q, head_dim=64, out=forward_ad.make_dual(out.detach(), torch.ones_like(out)))
    assert torch.equal(out, keep)
    with torch.no_grad():
        block.attention(q, q, q, head_dim=64, out=out)
    assert torch.equal(out, block.attention(q, q, q, head_dim=64))


# ---- arguments that share memory
def test_rotary_in_place_refuses_shared_memory():
    wide = randn(20, 512)
    for q, k in ((wide, wide), (wide[:, :128], wide[:, 64:192]), (wide[:10], wide[:10]), (wide[:, :128], wide[:, :64]),
                 (wide[0:1, :128], wide[0:1, 64:192])):
        with pytest.raises(ValueError, match="share memory"):
            block.rotary_(q, k, SPEC, head_dim=64)
    keep = wide.clone()
    block.rotary_(wide[:, :128], wide[:, 128:192], SPEC, head_dim=64)  # side by side
    block.rotary_(wide[:10, 192:256], wide[10:, 192:256], SPEC, head_dim=64)  # one above the other
    assert torch.equal(wide[:, 256:], keep[:, 256:])
    turned, _ = block.rotary(keep[:, :128], None, SPEC, head_dim=64)
    assert torch.equal(wide[:, :128], turned)
    same, again = block.rotary(keep, keep, SPEC, head_dim=64)  # read twice is fine
    assert torch.equal(same, again)


def test_attention_refuses_an_output_over_an_input():
    wide = randn(64, 512)
    q, k, v = wide[:, :128], wide[:, 128:192], wide[:, 192:256]
    for out in (q, wide[:, 64:192], wide[:, 192:320]):
        with pytest.raises(ValueError, match="share memory"):
            block.attention(q, k, v, head_dim=64, out=out)
    want = block.attention(q, k, v, head_dim=64)
    block.attention(q, k, v, head_dim=64, out=wide[:, 256:384])  # beside them
    assert torch.equal(wide[:, 256:384], want)


# ---- numbers past 31 bits
def test_numbers_past_31_bits_are_refused():
    q = randn(300, 64)
    for kw in (dict(window=(1 << 32) + 5), dict(window=1 << 31), dict(window=5, sinks=1 << 32), dict(q_len=(1 << 32) + 300), dict(kv_len=(1 << 32) + 300)):
        with pytest.raises(ValueError):
            block.attention(q, q, q, head_dim=64, **kw)
    whole = block.attention(q, q, q, head_dim=64)
    assert torch.equal(block.attention(q, q, q, head_dim=64, window=(1 << 31) - 1, sinks=(1 << 31) - 1), whole)
    with pytest.raises(ValueError):
        block.rotary(q, None, block.Rotary((1 << 32) + 64), head_dim=64)
    for kw in (dict(seq_len=(1 << 64) + 300), dict(start=1 << 63)):
        with pytest.raises(ValueError):
            block.rotary(q, None, SPEC, head_dim=64, **kw)


# ---- the norm that gives both forms at once has the gradient of the one that gives BF16
@pytest.mark.parametrize("rows,hidden", [(1, 32), (130, 1024), (33, 5120), (5, 8224)])
def test_gradient_beside_the_mxfp8_form(rows, hidden):
    x, residual, gamma, dy, dh = randn(rows, hidden, seed=1), randn(rows, hidden, seed=2), randn(hidden, seed=3), randn(rows, hidden, seed=4), randn(rows, hidden, seed=5)
    results = []
    for mxfp8 in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, residual, gamma)]
        y, h, *packed = block.rms_norm(leaves[0], leaves[2], leaves[1], mxfp8=mxfp8)
        assert all(not t.requires_grad for t in packed)
        results.append((y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh))))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    h2, data, scales = block.rms_norm_mxfp8(x, gamma, residual)
    assert torch.equal(h2, results[1][1]) and torch.equal(data, packed[0]) and torch.equal(scales, packed[1])


# ---- a refusal names its reason
def test_refusals_name_their_reason():
    x, gamma, q = randn(8, 512), randn(512), randn(8, 128)
    odd = randn(8, 136)[:, :128].as_strided((7, 128), (132, 1))
    for call, words in (
            (lambda: block.rms_norm(x[:, 4:260], gamma[:256]), "x is not on a 16-byte boundary"),
            (lambda: block.rms_norm(x[:, :256], gamma[4:260]), "gamma is not on a 16-byte boundary"),
            (lambda: block.rms_norm(x[:, :252], gamma[:252]), "hidden is a multiple of 8"),
            (lambda: block.rms_norm(x, gamma, eps=0.0), "eps"),
            (lambda: block.rotary(q, None, block.Rotary(128), head_dim=64), "rotary_dim"),
            (lambda: block.rotary(q, None, block.Rotary(64, scaling="yarn", factor=2.0), head_dim=64), "scaling"),
            (lambda: block.attention(q, q, q, head_dim=32), "head_dim is 64 or 128"),
            (lambda: block.attention(q, q, q, head_dim=64, scale=0.0), "scale"),
            (lambda: block.attention(q, q, q, head_dim=64, q_len=9), "rows are in q"),
            (lambda: block.attention(q, q, q, head_dim=64, kv_len=9), "rows are in k"),
            (lambda: block.attention(q, q, q, head_dim=64, q_len=-1), "not negative"),
            (lambda: block.attention(odd, q[:7], q[:7], head_dim=64), "q's rows are 132 elements apart")):
        with pytest.raises(RuntimeError, match=words):
            call()
