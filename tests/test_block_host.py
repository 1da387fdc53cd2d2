"""CPU-side checks of the block operators (include/fuse_b200.h: RMS norm, rotary positions): what they refuse
before they touch a device, and the rotary frequencies against the formulas in 64 bits."""
import math

import pytest
import torch

from fuse_b200 import _native as N
from fuse_b200 import api, block

PTR = 1 << 20  # never dereferenced: every call below is refused on the host
INVALID = N.CUDA_ERROR_INVALID_VALUE


def norm_params(**kw):
    p = N.RmsNormParams(input=PTR, gamma=PTR, output=PTR, input_stride=-1, residual_stride=-1, residual_output_stride=-1,
                        output_stride=-1, rows=4, hidden=256, epsilon=1e-6)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(hidden=0), dict(hidden=12), dict(hidden=16392), dict(epsilon=0.0), dict(epsilon=-1.0), dict(epsilon=math.inf),
    dict(epsilon=math.nan), dict(output=None), dict(input=None), dict(input=PTR + 2), dict(gamma=None), dict(gamma=PTR + 8),
    dict(input_stride=248), dict(input_stride=260), dict(residual=PTR + 4), dict(residual=PTR, residual_stride=8),
    dict(residual_output=PTR + 8), dict(output_stride=255), dict(hidden=264, quantized=N.Mxfp8Activation(data=PTR, scales=PTR)),
    dict(quantized=N.Mxfp8Activation(data=PTR, scales=PTR, data_bytes=1023, scale_bytes=1024)),
    dict(quantized=N.Mxfp8Activation(data=PTR, scales=PTR, data_bytes=1024, scale_bytes=1023)),
    dict(quantized=N.Mxfp8Activation(data=PTR, scales=None, data_bytes=1024, scale_bytes=1024)),
])
def test_rms_norm_refuses(bad):
    assert api.launch_rms_norm(norm_params(**bad)) == INVALID


def test_rms_norm_takes_what_it_documents():
    # validation passes; without a device the call then says so, with another code
    for good in (dict(), dict(residual=PTR, residual_output=PTR), dict(input_stride=264), dict(hidden=16384),
                 dict(output=None, quantized=N.Mxfp8Activation(data=PTR, scales=PTR, data_bytes=1024, scale_bytes=1024))):
        if not torch.cuda.is_available():
            assert api.launch_rms_norm(norm_params(**good)) not in (0, INVALID)
    assert api.launch_rms_norm(norm_params(rows=0)) == 0
    assert N.lib().fuse_b200_launch_rms_norm(None, None) == INVALID


def norm_backward_params(**kw):
    p = N.RmsNormBackwardParams(grad_output=PTR, stream_input=PTR, gamma=PTR, grad_input=PTR, grad_output_stride=-1,
                                stream_input_stride=-1, grad_stream_stride=-1, grad_input_stride=-1, rows=4, hidden=256,
                                epsilon=1e-6)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(hidden=4), dict(hidden=16392), dict(epsilon=math.nan), dict(grad_output=None), dict(stream_input=PTR + 2),
    dict(gamma=None), dict(grad_input=None), dict(grad_stream=PTR + 2), dict(grad_stream=PTR, grad_stream_stride=128),
    dict(grad_output_stride=0), dict(grad_input_stride=257), dict(grad_gamma=PTR + 1),
])
def test_rms_norm_backward_refuses(bad):
    assert api.launch_rms_norm_backward(norm_backward_params(**bad)) == INVALID


def test_rms_norm_backward_workspace_refuses():
    for rows, hidden in ((-1, 256), (4, 0), (4, 12), (4, 16392)):
        assert api.rms_norm_backward_workspace_size(rows, hidden)[0] == INVALID
    assert N.lib().fuse_b200_rms_norm_backward_workspace_size(4, 256, None) == INVALID


def rotary_params(**kw):
    p = N.RotaryParams(q=PTR, k=PTR, q_output=PTR, k_output=PTR, q_stride=-1, k_stride=-1, q_output_stride=-1,
                       k_output_stride=-1, rows=4, seq_len=4, spec=block.Rotary(128).record(), q_heads=4, kv_heads=1,
                       head_dim=128)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


@pytest.mark.parametrize("bad", [
    dict(head_dim=126), dict(head_dim=0), dict(q_heads=-1), dict(q_heads=0, kv_heads=0), dict(rows=-1), dict(seq_len=0),
    dict(q=None), dict(q_output=None), dict(k=PTR + 1), dict(k_stride=127), dict(q_output_stride=256),
    dict(q_stride=1024), dict(positions=PTR), dict(positions=PTR, position_bytes=2), dict(positions=PTR + 4, position_bytes=8),
    dict(spec=block.Rotary(127).record()), dict(spec=block.Rotary(0).record()), dict(spec=block.Rotary(258).record()),
    dict(spec=block.Rotary(128, theta=0.0).record()), dict(spec=block.Rotary(128, theta=math.inf).record()),
    dict(spec=block.Rotary(128, scaling="linear", factor=0.0).record()),
    dict(spec=block.Rotary(2, scaling="ntk", factor=2.0).record()),
    dict(spec=block.Rotary(128, scaling="yarn", factor=2.0).record()),  # no original context
    dict(spec=block.Rotary(128, scaling="wavelength", factor=2.0, original_context=8, low_freq_factor=4.0).record()),
    dict(spec=block.Rotary(128, scaling="yarn", factor=2.0, original_context=8, beta_fast=1.0).record()),
    dict(spec=block.Rotary(128, magnitude=-1.0).record()),
])
def test_rotary_refuses(bad):
    assert api.launch_rotary(rotary_params(**bad)) == INVALID


def test_rotary_refuses_unknown_scaling():
    spec = block.Rotary(128).record()
    spec.scaling = 5
    assert api.rotary_frequencies(spec)[0] == INVALID
    assert api.launch_rotary(rotary_params(rows=0)) == 0
    with pytest.raises(ValueError):
        block.Rotary(128, scaling="cubic").record()
    with pytest.raises(ValueError):
        block.Rotary(7).frequencies()


@pytest.mark.parametrize("dim", [2, 64, 128, 256])
def test_rotary_frequencies(dim):
    theta, half = 500000.0, dim // 2
    base = [theta ** (-2.0 * i / dim) for i in range(half)]

    def close(spec, want, magnitude=1.0):
        values, m = spec.frequencies()
        assert m == pytest.approx(magnitude, rel=1e-15)
        assert values == pytest.approx(want, rel=1e-13)

    close(block.Rotary(dim, theta), base)
    close(block.Rotary(dim, theta, magnitude=0.5), base, 0.5)
    close(block.Rotary(dim, theta, scaling="linear", factor=4.0), [f / 4 for f in base])
    if dim > 2:
        stretched = theta * 4.0 ** (dim / (dim - 2))
        close(block.Rotary(dim, theta, scaling="ntk", factor=4.0), [stretched ** (-2.0 * i / dim) for i in range(half)])
    want = []
    for f in base:
        wavelength = 2 * math.pi / f
        if wavelength > 8192 / 1.0:
            want.append(f / 8)
        elif wavelength < 8192 / 4.0:
            want.append(f)
        else:
            keep = (8192 / wavelength - 1.0) / 3.0
            want.append((1 - keep) * f / 8 + keep * f)
    close(block.Rotary(dim, theta, scaling="wavelength", factor=8.0, original_context=8192), want)
    at = [dim * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
    want = []
    for i, f in enumerate(base):
        ramp = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
        want.append(f * (1 - ramp) + f / 16 * ramp)
    close(block.Rotary(dim, theta, scaling="yarn", factor=16.0, original_context=8192), want, 0.1 * math.log(16.0) + 1)


def test_torch_arguments_are_refused():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    g = torch.ones(256, dtype=torch.bfloat16)
    for call in (lambda: block.rms_norm(x, g), lambda: block.rms_norm(x.float(), g), lambda: block.rms_norm_mxfp8(x, g),
                 lambda: block.rotary(x, None, block.Rotary(128), head_dim=128),
                 lambda: block.rotary(None, None, block.Rotary(128), head_dim=128)):
        with pytest.raises(ValueError):
            call()


def attention_params(**kw):
    p = N.AttentionParams(q=PTR, k=PTR, v=PTR, output=PTR, q_stride=-1, k_stride=-1, v_stride=-1, output_stride=-1, q_rows=256,
                          kv_rows=512, batch=2, q_len=128, kv_len=256, q_heads=8, kv_heads=2, head_dim=128, causal=1, scale=0.1)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


SHAPE_FAULTS = [
    dict(batch=-1), dict(q_len=-1), dict(kv_len=-1), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=7), dict(window=-1), dict(sinks=-1),
    dict(causal=0, window=4), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(q_len=129),
    dict(kv_len=257), dict(q_rows=-1), dict(q_rows=2 ** 31), dict(kv_rows=2 ** 31), dict(q_len=2 ** 30, q_starts=PTR),
]
POINTER_FAULTS = [
    dict(q=None), dict(q=PTR + 8), dict(k=None), dict(v=PTR + 2), dict(output=None), dict(output_stride=1020), dict(q_stride=1028),
    dict(k_stride=128), dict(v_stride=252), dict(lse=PTR + 2),
]


@pytest.mark.parametrize("bad", SHAPE_FAULTS + POINTER_FAULTS)
def test_attention_refuses(bad):
    assert api.launch_attention(attention_params(**bad)) == INVALID


@pytest.mark.parametrize("bad", SHAPE_FAULTS)
def test_attention_workspace_refuses(bad):
    assert api.attention_workspace_size(attention_params(**bad))[0] == INVALID
    assert api.attention_backward_workspace_size(N.AttentionBackwardParams(forward=attention_params(**bad)))[0] == INVALID


def attention_backward_params(**kw):
    forward = {key: kw.pop(key) for key in list(kw) if hasattr(N.AttentionParams, key) and key not in ("workspace", "workspace_bytes")}
    p = N.AttentionBackwardParams(forward=attention_params(**{"lse": PTR, **forward}), grad_output=PTR, grad_q=PTR, grad_k=PTR,
                                  grad_v=PTR, grad_output_stride=-1, grad_q_stride=-1, grad_k_stride=-1, grad_v_stride=-1,
                                  workspace=PTR, workspace_bytes=1 << 30)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


@pytest.mark.parametrize("bad", SHAPE_FAULTS + POINTER_FAULTS + [
    dict(lse=None), dict(grad_output=None), dict(grad_q=PTR + 8), dict(grad_k=None), dict(grad_v=None), dict(grad_q_stride=512),
    dict(grad_k_stride=260), dict(grad_output_stride=8), dict(workspace=None), dict(workspace=PTR + 128), dict(workspace_bytes=8 * 256 * 4 - 1),
])
def test_attention_backward_refuses(bad):
    assert api.launch_attention_backward(attention_backward_params(**bad)) == INVALID


def test_attention_without_work_or_support():
    assert api.launch_attention(attention_params(head_dim=96)) == N.CUDA_ERROR_NOT_SUPPORTED
    assert api.launch_attention(attention_params(batch=0, q=None)) == 0
    assert api.launch_attention(attention_params(q_len=0, q=None)) == 0
    assert api.launch_attention_backward(attention_backward_params(batch=0)) == 0
    assert N.lib().fuse_b200_launch_attention(None, None, None) == INVALID
    assert N.lib().fuse_b200_launch_attention_backward(None, None, None) == INVALID
