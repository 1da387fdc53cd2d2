"""Calls from several host threads at once (autograd has threads of its own): one call's launch does not change another's."""
import threading

import pytest
import torch

from fuse_b200 import _native as N
from fuse_b200 import api

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def test_norm_backward_of_different_widths_from_two_threads():
    rows, calls = 2, 4000
    failures = []

    def work(hidden):
        torch.cuda.set_device(0)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            dy, h, dx = (torch.ones(rows, hidden, dtype=BF16, device=DEV) for _ in range(3))
            gamma = torch.ones(hidden, dtype=BF16, device=DEV)
            p = N.RmsNormBackwardParams(grad_output=dy.data_ptr(), stream_input=h.data_ptr(), gamma=gamma.data_ptr(), grad_input=dx.data_ptr(),
                                        grad_output_stride=-1, stream_input_stride=-1, grad_stream_stride=-1, grad_input_stride=-1,
                                        rows=rows, hidden=hidden, epsilon=1e-6)
            for i in range(calls):
                rc = api.launch_rms_norm_backward(p, stream.cuda_stream)
                if rc != 0:
                    failures.append((hidden, i, rc))
                    break
                if i % 256 == 255:
                    stream.synchronize()
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(hidden,)) for hidden in (1024, 16384, 5120, 16384)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert failures == []
