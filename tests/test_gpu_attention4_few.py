"""Which kernel takes a sequence of few rows over a cache of 4 bits: a draft is not slower than one of a token more.

Streaming goes by tiles of whole tokens, 8 rows each: with three to seven query heads to a key head that do not fill them, a rule that counts rows streams five or six tiles (32 drafts of six tokens
of 5 heads 189 us, of seven, on the tensor cores, about 140)."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_attention4 import check, forward  # noqa: E402
from test_gpu_kv4 import Cache4, backend, stream  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def call_time(b, c):
    """us of a call, the least of some captured ones."""
    forward(b, c)
    batch, side, graph = c.batch(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        for _ in range(10):
            b.attention_forward_device(0, batch, c.q.data_ptr(), c.out.data_ptr(), side.cuda_stream, q_stride=c.q_all.stride(0))
    times = []
    for _ in range(10):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end) * 100)
    b.stream_check(0, stream())
    return min(times)


@pytest.mark.parametrize("group,longest", [(3, 12), (4, 9), (5, 7), (6, 6), (7, 5), (8, 5), (12, 5)])
def test_more_tokens_are_not_faster(backend, group, longest):  # noqa: F811
    times = []
    for n in range(1, longest + 1):
        c = Cache4([(n, 3000 + n + 50 * i) for i in range(32)], 8 * group, 8, 128, "bf16", 16).install(backend)
        for p in c.pools:
            p.zero_()
        times.append(call_time(backend, c))
    assert all(a <= 1.1 * b for a, b in zip(times, times[1:])), times


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16, 17])
def test_drafts_beside_the_border(backend, group):  # noqa: F811
    for n in sorted({n for rows in (15, 18, 24, 32, 36, 48) for n in (rows // group, rows // group + 1) if n}):
        c = Cache4([(n, 300 + n), (1, 130), (n, n), (max(1, n - 1), 500)], 2 * group, 2, 64, "bf16", 16, behind=2).fill().install(backend)
        forward(backend, c)
        backend.stream_check(0, stream())
        check(c)
