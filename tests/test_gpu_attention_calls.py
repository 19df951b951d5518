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


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 40), (1, 3), (1, 9000)], [(40, 40), (300, 700), (2, 3), (5, 6000)]])
def test_sinks_of_minus_infinity(backend, lens, d):  # noqa: F811
    """A head whose sink is -infinity has none; beside scores that are all -infinity its rows attend to nothing."""
    c = Cache(lens, 8, 2, d, "bf16", 16).fill()
    sinks = np.array([-math.inf, 1.0, -math.inf, 0.0, -math.inf, -2.0, 3.0, -math.inf], np.float32)
    c.install(backend, sinks=sinks)
    c.forward(backend)
    c.check()
    c.q.view(-1, 8, d)[:, :, 0] = c.q.view(-1, 8, d)[:, :, 0].abs() + 0.5
    for i, (n, k) in enumerate(lens):
        c.k[(*c.places(i), 0, 0)] = -math.inf  # every token of the first key head: heads 0 .. 3
    c.forward(backend)
    out = c.out.view(-1, 8, d)
    assert (out[:, :4] == 0).all()
    # the other key head's queries have new first values: against its own formula
    u = torch.finfo(c.kind).eps / 2
    for i, (n, k) in enumerate(lens):
        keys, values = (x[c.places(i)][:, 1].double() for x in (c.k, c.v))
        q = c.q[c.starts[i]:c.starts[i + 1]].double().view(n, 8, d)[:, 4:].transpose(0, 1)
        s = q @ keys.T * d ** -0.5
        size = (q.abs() @ keys.abs().T * d ** -0.5).amax(2, keepdim=True)
        hidden = torch.arange(k, device="cuda") > torch.arange(k - n, k, device="cuda")[:, None]
        s = s.masked_fill(hidden, -math.inf)
        total = torch.logaddexp(torch.logsumexp(s, 2, keepdim=True), torch.tensor(sinks[4:], dtype=torch.float64, device="cuda")[:, None, None])
        p = (s - total).exp()
        want, a = p @ values, p @ values.abs()
        bound = u * (a + want.abs()) * 1.01 + (2 * size * (d + 3) * 2.0 ** -24 + 2.0 ** -18) * a + 2.0 ** -24
        got = out[c.starts[i]:c.starts[i + 1], 4:].double().transpose(0, 1)
        assert ((got - want).abs() <= bound).all()


def test_a_sink_that_is_not_a_number_is_refused(backend):  # noqa: F811
    sinks = np.zeros(8, np.float32)
    sinks[5] = math.nan
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.install_attention(9, 8, 2, 64, mer_b200.VALUE_F16, 16, sinks=sinks)
    assert e.value.kind == INVALID


def test_first_calls_on_a_stream_of_their_own(backend):  # noqa: F811
    """A layer is ready when its installation returns, on streams too that do not wait for the one its constants were copied on."""
    d, stream = 256, torch.cuda.Stream()
    c = Cache([(1, 40), (1, 900)], 8, 2, d, "bf16", 16).fill()
    x = torch.randn((2, 12 * d), device="cuda")
    weights, freq, sinks = np.linspace(0.5, 1.5, d).astype(np.float32), 1e4 ** (-np.arange(d // 2) * 2 / d), np.linspace(-2, 2, 8).astype(np.float32)
    outs = [torch.zeros((2, 8 * d), device="cuda", dtype=c.kind) for _ in range(31)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        # every installation is the first one of its layer, in memory that held other constants
        with mer_b200.Backend(mer_b200.DTYPE_Q8_0, 64, 64, 1 << 20, 1, max_tokens=1, max_top_k=1) as b:
            b.install_attention(1, 8, 2, d, c.value_type, 16, q_norm=-7 * weights, k_norm=weights + 3, rope_freq=freq[::-1], sinks=sinks + 5)
            b.install_attention(2, 8, 2, d, c.value_type, 16, q_norm=weights, k_norm=weights, rope_freq=freq, sinks=sinks)
            rows = mer_b200.QkvRows(q=x.data_ptr(), k=x.data_ptr() + 4 * 8 * d, v=x.data_ptr() + 4 * 10 * d, q_out=c.q.data_ptr(), q_stride=12 * d, k_stride=12 * d,
                                    v_stride=12 * d, value_type=mer_b200.VALUE_F32)
            b.kv_append_device(2, c.batch(), rows, stream.cuda_stream)
            b.attention_forward_device(2, c.batch(), c.q.data_ptr(), out.data_ptr(), stream.cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(out, outs[0]), i
    c.opts = dict(sinks=sinks)
    c.check(torch.cat([outs[0], c.out[2:]]))


SINGLE, SEVERAL = [(1, 100), (1, 900), (1, 60)], [(1, 100), (6, 900), (70, 75)]  # one row a sequence: the streaming kernel; more: the other one


@pytest.mark.parametrize("lens", [SINGLE, SEVERAL])
@pytest.mark.parametrize("page", [16, 5])  # with tiled copies, and row by row
@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (128, 300), (256, 0)])
def test_tokens_without_a_page_count_as_zeros(backend, lens, page, d, window):  # noqa: F811
    c = Cache(lens, 8, 2, d, "bf16", page).fill().install(backend, window=window)
    stands = Cache(lens, 8, 2, d, "bf16", page)  # the same with zeros in those places
    stands.k, stands.v, stands.q, stands.table, stands.opts = c.k.clone(), c.v.clone(), c.q, c.table.clone(), c.opts
    held = -(-lens[1][1] // page)
    for slot, number in ((2, c.n_pages), (held // 2, -1), (held - 3, 0x7FFFFFFF), (held - 2, c.n_pages + 1)):
        first, last = slot * page, min(slot * page + page, lens[1][1])
        for x in (stands.k, stands.v):
            x[stands.places(1, first, last)] = 0.0
        c.table[1, slot] = number
    c.forward(backend)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.stream_check(0, current())
    assert e.value.kind == DISPATCH
    stands.check(c.out)


@pytest.mark.parametrize("lens", [SINGLE, SEVERAL])
@pytest.mark.parametrize("page,d", [(16, 64), (5, 64), (16, 128), (16, 256)])
def test_values_that_are_not_finite_stay_in_their_sequence_and_head(backend, lens, page, d):  # noqa: F811
    c = Cache(lens, 8, 2, d, "bf16", page).fill().install(backend)
    good = c.forward(backend).clone().view(-1, 8, d)
    pages, slots = c.places(1)
    a, b = c.starts[1], c.starts[2]
    c.v[pages[850], slots[850], 1, 5] = math.inf
    c.forward(backend)
    out = c.out.clone().view(-1, 8, d)
    assert not torch.isfinite(out[a:b, 4:, 5]).any()  # the first value of its group's heads that every row sees
    out[a:b, 4:, 5] = good[a:b, 4:, 5]
    assert torch.equal(out, good)
    c.k[pages[20], slots[20], 0, 3] = math.nan
    c.forward(backend)
    out = c.out.view(-1, 8, d)
    assert torch.isnan(out[a:b, :4]).all()
    assert torch.equal(out[:a], good[:a]) and torch.equal(out[b:], good[b:])


@pytest.mark.parametrize("lens", [[(1, 200), (1, 170), (1, 2000), (1, 129)], [(5, 200), (40, 170), (1, 2000), (3, 131)]])
@pytest.mark.parametrize("page", [16, 5])
def test_sequences_that_share_the_pages_of_their_beginning(backend, lens, page):  # noqa: F811
    c = Cache(lens, 8, 2, 128, "f16", page)
    shared = 100 // page
    c.table[1:, :shared] = c.table[0, :shared]
    c.fill().install(backend)
    before = c.k.clone()
    x = torch.randn((c.rows, 12 * 128), device="cuda", dtype=c.kind)
    at = x.data_ptr()
    rows = mer_b200.QkvRows(q=at, k=at + 2048, v=at + 2560, q_out=c.q.data_ptr(), q_stride=1536, k_stride=1536, v_stride=1536, value_type=c.value_type)
    backend.kv_append_device(0, c.batch(), rows, current())  # no norms, no rotation: as they are
    c.forward(backend)
    backend.stream_check(0, current())
    assert torch.equal(c.k[c.table[0, :shared].long()], before[c.table[0, :shared].long()])
    for i, (n, k) in enumerate(lens):
        assert torch.equal(c.k[c.places(i, k - n)].flatten(1), x[c.starts[i]:c.starts[i + 1], 1024:1280])
    assert torch.equal(c.q, x[:, :1024])
    c.check()
