"""Appending to a cache of 4 bits: a step of keys holds as many heads as a warp's lanes have room for, and a step that some of them do not fill is as fast as a full one.

In 64 bits, where a step goes whose 32-bit values lie too near a border, it takes far longer: with every step that is not full made there, 11000 rows of one key head of 128 took 32.4 us and of
two 25.3, of three key heads of 80 47.6 and of four 40.8."""
import pytest

import mer_b200

torch = pytest.importorskip("torch")
from test_gpu_kv4 import Cache4, append, backend, stream  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def append_time(b, c):
    """us of an append of the batch's rows, the least of some captured ones."""
    append(b, c, "bf16", rope_dims=c.d // 2 // 8 * 8)
    width = (c.hq + 2 * c.hk) * c.d
    x = torch.randn(c.rows, width, device="cuda", generator=c.gen).bfloat16()
    at = x.data_ptr()
    rows = mer_b200.QkvRows(q=None, k=at + c.hq * c.d * 2, v=at + (c.hq + c.hk) * c.d * 2, k_stride=width, v_stride=width, value_type=mer_b200.VALUE_BF16)
    batch, side, graph = c.batch(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        for _ in range(10):
            b.kv_append_device(0, batch, rows, side.cuda_stream)
    times = []
    for _ in range(12):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end) * 100)
    b.stream_check(0, stream())
    return min(times)


@pytest.mark.parametrize("d,some,full", [(128, 1, 2), (80, 3, 4), (64, 1, 4), (64, 7, 8)])
def test_steps_that_heads_do_not_fill(backend, d, some, full):  # noqa: F811
    lens = [(6000, 6000), (5000, 7000)]
    few, many = (append_time(backend, Cache4(lens, h, h, d, "bf16", 16)) for h in (some, full))
    assert few <= 1.1 * many, (few, many)
