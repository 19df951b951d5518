"""Calls of the attention side that follow one another without a wait, and layers, tables and values at the edge of what the header allows."""
import math

import numpy as np
import pytest

import mer_b200
from test_gpu_attention import DISPATCH, INVALID, Cache, backend  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def current():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("lens", [[(1, 20 + i % 70) for i in range(300)], [(1 + i % 5, 30 + i) for i in range(90)]])
@pytest.mark.parametrize("d,offset,gap", [(64, 8, 8), (24, 0, 16), (128, 24, 0)])
def test_append_in_place_and_attention_right_behind_it(backend, lens, d, offset, gap):  # noqa: F811
    """Rows that start on 16 bytes but not on 128: the heads of two rows, which different SMs rotate, share lines that the next call reads whole."""
    hq, hk = 8, 2
    c = Cache(lens, hq, hk, d, "bf16", 16).fill()
    c.install(backend, 0, q_norm=np.linspace(0.5, 1.5, d).astype(np.float32), rope_freq=1e4 ** (-np.arange(d // 2) * 2 / d))
    width = (hq + 2 * hk) * d + gap
    store = torch.randn(c.rows * width + offset, device="cuda").to(c.kind)
    want = work = None
    for wait in (True, False):
        for _ in range(1 if wait else 40):
            work = store.clone()
            x = work[offset:].view(c.rows, width)
            at = x.data_ptr()
            rows = mer_b200.QkvRows(q=at, k=at + 2 * hq * d, v=at + 2 * (hq + hk) * d, q_out=at, q_stride=width, k_stride=width, v_stride=width, q_out_stride=width,
                                    value_type=c.value_type)
            out = torch.full_like(c.out, 7.0)
            backend.kv_append_device(0, c.batch(), rows, current())
            if wait:
                torch.cuda.synchronize()
            backend.attention_forward_device(0, c.batch(), at, out.data_ptr(), current(), q_stride=width)
            if wait:
                torch.cuda.synchronize()
                want = out
                c.q = x[:, :hq * d].clone()
                c.check(out)
            else:
                assert torch.equal(out, want)
    backend.stream_check(0, current())
