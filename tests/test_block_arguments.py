"""Host arithmetic behind the block operators' refusals (fuse_b200/block.py)."""
import random

import pytest
import torch

from fuse_b200 import api, block
from tests.test_block_host import INVALID, PTR, attention_backward_params, attention_params


def test_overlap_of_row_views_against_enumeration():
    base = torch.arange(400, dtype=torch.int32)
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        views = []
        pitch = rng.choice((7, 12, 20))
        for _ in range(2):
            if rng.random() < 0.2:
                pitch = rng.choice((7, 12, 20))
            rows, width = rng.randint(1, 5), rng.randint(1, pitch)
            views.append(base.as_strided((rows, width), (pitch, 1), rng.randint(0, 200)))
        a, b = views
        want = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert block._overlap(a, b) == block._overlap(b, a) == want, (a, b)
        seen[want] += 1
    assert min(seen.values()) > 1000
    assert not block._overlap(base[:0].view(0, 4), base.view(100, 4))
    half = base.view(torch.bfloat16).view(100, 8)
    assert block._overlap(half[:, :4], half[:, 3:]) and not block._overlap(half[:, :4], half[:, 4:])


def test_numbers_that_a_record_would_cut_off():
    block._within(32, window=(1 << 31) - 1, sinks=-(1 << 31))
    block._within(64, start=(1 << 63) - 1)
    for bits, value in ((32, 1 << 31), (32, (1 << 32) + 5), (32, -(1 << 31) - 1), (64, 1 << 63), (64, (1 << 64) + 300)):
        with pytest.raises(ValueError, match="window: "):
            block._within(bits, window=value)
    with pytest.raises(ValueError, match="rotary_dim"):
        block.Rotary((1 << 32) + 64).record()
    with pytest.raises(ValueError, match="original_context"):
        block.Rotary(64, scaling="yarn", factor=2.0, original_context=(1 << 64) + 8192).frequencies()


def test_attention_refuses_an_unaligned_rest():
    p = attention_params(output_rest=PTR + 8)
    assert api.launch_attention(p) == INVALID
    assert api.launch_attention_backward(attention_backward_params(output_rest=PTR + 8)) == INVALID
    if not torch.cuda.is_available():  # an aligned one passes the checks and meets the missing device
        assert api.launch_attention(attention_params(output_rest=PTR + 16)) not in (0, INVALID)
