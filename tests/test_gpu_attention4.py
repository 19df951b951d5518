"""Attention over a paged cache of 4 bits (mer_attention_forward_device of a layer whose cache holds 4 bits) against the formulas in 64 bits, on
the values that codes, scales and minima stand for.

Bounds.  A rounding to a type is off by at most u = eps / 2 of the value.  The kernels' operands are f16 (u16 = 2^-11): a key is scale * code +
minimum rounded once, or exact codes with scale and minimum in fp32; a weight is rounded once, a value is, or a weight times a scale is rounded
once more: at most 3 u16 of V = sum_j p_j (scale code + |minimum|).  A score is off by at most u16 + (D + 3) 2^-24 of S = scale sum |q| (scale code +
|minimum|), and by 2^-24 of a row's largest query times what it multiplies (queries are held as f16 beside their row's power of two); that moves a weight, and the sum
that it is divided by, by as much in proportion.  Exponentials, sums and joins add less than 2^-18 of V; the output is rounded once, u * |o|."""
import math

import numpy as np
import pytest

import mer_b200

torch = pytest.importorskip("torch")
from test_gpu_kv4 import DISPATCH, LENS as ROWS, Cache4, append, backend, numbers, quantised, read, stream  # noqa: E402, F401

pytestmark = pytest.mark.gpu
U16 = 2.0 ** -11

LENS = {
    "one": [(1, 1)],
    "decode": ROWS["decode"],
    "long": [(1, 9000)],
    "idle": ROWS["idle"],
    "draft": [(5, 70), (3, 3), (7, 513), (2, 1025)],
    "prompts": ROWS["prompts"],
    "chunk": [(300, 1500)],
}


def forward(b, c, layer=0, **kw):
    b.attention_forward_device(layer, c.batch(**kw), c.q.data_ptr(), c.out.data_ptr(), stream(), q_stride=c.q_all.stride(0))
    return c.out


def magnitudes(c, keys, places):
    """scale * code + |minimum| of what the cache has there."""
    words, pairs = c.parts(keys)
    held = c.held(keys, places)
    least = pairs[places[0], :, places[1]].double()[..., 1][..., torch.arange(c.d, device="cuda") // c.group]
    return held - least + least.abs()


def check(c, out=None):
    out = c.out if out is None else out
    u, window, g = torch.finfo(c.kind).eps / 2, c.opts.get("window", 0), c.hq // c.hk
    scale = c.opts.get("scale", 0) or c.d ** -0.5
    sinks = c.opts.get("sinks")
    for i, (n, k) in enumerate(c.lens):
        if n == 0 or k == 0:
            continue
        pos = torch.arange(k - n, k, device="cuda")
        lo = max(0, k - n - window + 1) if window else 0  # what is before it may be anything
        at = torch.arange(lo, k, device="cuda")
        places = c.places(i, lo)
        keys, values, big_k, big_v = (f(*a).transpose(0, 1) for f in (c.held, lambda x, y: magnitudes(c, x, y)) for a in ((True, places), (False, places)))
        q = c.q[c.starts[i]:c.starts[i + 1]].double().view(n, c.hk, g, c.d).permute(1, 2, 0, 3)
        s = torch.einsum("hgnd,htd->hgnt", q, keys) * scale
        size = torch.einsum("hgnd,htd->hgnt", q.abs(), big_k) * scale * (U16 + (c.d + 3) * 2.0 ** -24)
        size += q.abs().amax(3, keepdim=True) * big_k.sum(2)[:, None, None] * scale * 2.0 ** -24
        hidden = at > pos[:, None]
        if window:
            hidden |= at <= pos[:, None] - window
        s = s.masked_fill(hidden, -math.inf)
        total = torch.logsumexp(s, 3, keepdim=True)
        if sinks is not None:
            total = torch.logaddexp(total, torch.tensor(sinks, dtype=torch.float64, device="cuda").view(c.hk, g, 1, 1))
        p = torch.where(hidden.all(1)[:, None], 0.0, (s - total).exp())
        want = torch.einsum("hgnt,htd->hgnd", p, values)
        a = torch.einsum("hgnt,htd->hgnd", p, big_v)
        move = torch.where(hidden, 0.0, size).amax(3, keepdim=True)  # only what a row sees moves its weights
        bound = u * want.abs() * 1.01 + (2 * move + 2.0 ** -18 + 3 * U16) * a * 1.01 + 2.0 ** -24
        got = out[c.starts[i]:c.starts[i + 1]].double().view(n, c.hk, g, c.d).permute(1, 2, 0, 3)
        worst = ((got - want).abs() / bound).max().item()
        assert worst <= 1.0, (i, n, k, worst)
        # rounded at random, the roundings of a row's values meet in their sum as their squares do: far below the bound on the whole
        spread = ((got - want).square().mean() / want.square().mean().clamp(min=1e-30)).sqrt().item()
        assert spread <= 2 * u + 8 * U16 or n * k < 200, (i, n, k, spread)
    assert (out[c.starts[-1]:] == 7.0).all()


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("q_heads,kv_heads,d,kind,page,group", [
    (8, 1, 128, "bf16", 16, 32), (32, 4, 128, "f16", 32, 64), (6, 6, 64, "bf16", 1, 32), (20, 4, 80, "f16", 24, 32), (2, 1, 8, "bf16", 3, 32), (40, 1, 64, "f16", 64, 64),
    (4, 2, 256, "bf16", 16, 32), (7, 1, 136, "f16", 5, 32), (2, 2, 8, "f16", 32, 64), (3, 1, 24, "bf16", 16, 32), (300, 1, 8, "f16", 16, 32), (130, 1, 200, "bf16", 128, 64),
    (1, 1, 256, "f16", 24, 64), (16, 1, 96, "bf16", 8, 64), (12, 1, 128, "f16", 40, 32), (10, 2, 192, "bf16", 16, 32), (16, 1, 256, "bf16", 256, 32), (9, 1, 160, "f16", 8, 64)])
def test_attention(backend, lens, q_heads, kv_heads, d, kind, page, group):  # noqa: F811
    c = Cache4(LENS[lens], q_heads, kv_heads, d, kind, page, group, behind=3).fill().install(backend)
    forward(backend, c)
    backend.stream_check(0, stream())
    check(c)


@pytest.mark.parametrize("lens", ["decode", "draft", "prompts", "chunk", "long"])
@pytest.mark.parametrize("window", [1, 2, 17, 128, 1000])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 32)])
def test_window_and_sinks(backend, lens, window, d, group):  # noqa: F811
    # tokens before every window are bytes of any kind, scales and minima that are not finite among them
    c = Cache4(LENS[lens], 8, 2, d, "bf16", 16, group, heads_first=True, seed=window, gap=48)
    c.fill([max(0, k - n - window + 1) for n, k in c.lens])
    c.install(backend, window=window, sinks=np.linspace(-3, 4, 8).astype(np.float32), scale=0.2)
    forward(backend, c)
    check(c)


@pytest.mark.parametrize("page", [1, 5, 8, 16, 24, 64])
def test_what_no_row_sees_may_be_anything(backend, page):  # noqa: F811
    # behind the last token of a page, and in pages of nobody: NaN scales and minima
    for lens in ([(1, 3), (1, 130), (1, 250)], [(4, 7), (40, 133), (1, 259)]):
        c = Cache4(lens, 8, 2, 128, "bf16", page, 32)
        for keys in (True, False):
            c.parts(keys)[1].fill_(math.nan)
        c.fill().install(backend)
        forward(backend, c)
        check(c)


def test_many_sequences(backend):  # noqa: F811
    rng = np.random.default_rng(5)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 4, 700), rng.integers(0, 200, 700))]
    c = Cache4(lens, 8, 2, 64, "f16", 8, seed=2, behind=5).fill().install(backend)
    forward(backend, c)
    check(c)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 2, 900), rng.integers(0, 400, 900))]
    c = Cache4(lens, 8, 2, 128, "bf16", 16, seed=2, behind=0).fill().install(backend)
    forward(backend, c)
    check(c)


@pytest.mark.parametrize("size", [1e-4, 3e-2, 40.0, 3000.0])
def test_values_of_any_size(backend, size):  # noqa: F811
    # keys and values far from one, and a token in sixty a hundred times as large
    for lens in ([(1, 700), (1, 40)], [(30, 700), (3, 40)]):
        c = Cache4(lens, 8, 2, 128, "f16", 16)
        for i, (n, k) in enumerate(lens):
            for keys in (True, False):
                x = torch.randn((k, 2, 128), device="cuda", generator=c.gen).double() * size
                x[7::60] *= 100.0 if size < 1000 else 5.0
                c.put(keys, c.places(i), *quantised(x, 32))
        c.q.mul_(0.5 / size)
        c.install(backend)
        forward(backend, c)
        u, out = torch.finfo(c.kind).eps / 2, c.out.double()
        assert torch.isfinite(out).all()
        check(c)


@pytest.mark.parametrize("page,d,group", [(5, 128, 32), (16, 80, 32), (24, 64, 64), (48, 256, 32)])
def test_large_values_in_tiles_behind_one_another(backend, page, d, group):  # noqa: F811
    # weights times scales that f16 has no room for, in some of the sequences that a CTA has one after the other, and not in others
    for lens in ([(1, 90 + i % 7) for i in range(900)], [(1 + i % 3, 400 + 50 * (i % 9)) for i in range(300)]):
        c = Cache4(lens, 8, 2, d, "bf16", page, group)
        for i, (n, k) in enumerate(lens):
            for keys in (True, False):
                size = 8000.0 if not keys and i % 5 == 2 else 1.0
                c.put(keys, c.places(i), *quantised(torch.randn((k, 2, d), device="cuda", generator=c.gen).double() * size, group))
        c.install(backend)
        forward(backend, c)
        check(c)


def test_queries_of_any_size(backend):  # noqa: F811
    for kind, sizes in (("bf16", (1e-30, 1e-5, 1e5)), ("f16", (1e-4, 300.0))):
        for lens in ([(1, 300), (1, 77)], [(30, 300), (3, 77)]):
            for size in sizes:
                c = Cache4(lens, 8, 2, 128, kind, 16, gap=16).fill(scale=min(1.0, 1 / size)).install(backend)
                c.q.mul_(size)
                c.q.view(-1, 8, 128)[:, 1] *= 2.0 ** -6  # a head's rows beside others far larger
                forward(backend, c)
                check(c)


def test_large_scores_and_small_weights(backend):  # noqa: F811
    # one key far above thousands of equal ones: what these sum to counts
    for lens in ([(1, 6000)], [(2, 6000)]):
        c = Cache4(lens, 4, 1, 64, "f16", 16).fill().install(backend)
        c.q.mul_(0).add_(1.0)
        x = torch.zeros((6000, 1, 64), dtype=torch.float64, device="cuda")
        x[3] = 10.0 * 8 / 64
        c.put(True, c.places(0), *quantised(x, 32))
        forward(backend, c)
        check(c)
        c.q.mul_(300.0)  # scores of thousands
        forward(backend, c)
        check(c)


def test_query_and_output_strides(backend):  # noqa: F811
    for lens in ("decode", "draft"):
        c = Cache4(LENS[lens], 8, 2, 64, "bf16", 16, q_gap=64).fill().install(backend)
        wide = torch.full((c.rows, 8 * 64 + 24), 3.0, dtype=c.kind, device="cuda")
        backend.attention_forward_device(0, c.batch(), c.q.data_ptr(), wide.data_ptr(), stream(), c.q_all.stride(0), wide.stride(0))
        check(c, wide[:, :512])
        assert (wide[:, 512:] == 3.0).all()


def test_keys_and_values_of_one_pool(backend):  # noqa: F811
    # [page][keys, values][head]
    for lens in ("decode", "chunk"):
        c = Cache4(LENS[lens], 8, 4, 128, "f16", 32)
        pool = torch.randint(0, 256, (c.n_pages, 2, 4, c.block), dtype=torch.uint8, device="cuda")
        c.k, c.v = pool[:, 0], pool[:, 1]
        c.fill().install(backend)
        forward(backend, c)
        check(c)


def test_same_bits_every_time(backend):  # noqa: F811
    for lens in ([(1, 5000), (3, 900), (40, 2000), (1, 2)], [(1, 5000), (1, 900), (1, 1), (1, 12000)]):
        c = Cache4(lens, 16, 2, 128, "bf16", 16).fill().install(backend)
        first = forward(backend, c).clone()
        for _ in range(20):
            assert torch.equal(forward(backend, c), first)


def test_sequence_with_more_rows_than_tokens(backend):  # noqa: F811
    for lens, kept, rows in (([(2, 50), (6, 4), (3, 0), (1, 20)], [(2, 50), (4, 4), (1, 20)], [0, 1, 4, 5, 6, 7, 11]), ([(1, 50), (1, 0), (1, 20)], [(1, 50), (1, 20)], [0, 2])):
        c = Cache4(lens, 8, 2, 64).fill().install(backend)
        forward(backend, c)
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            backend.stream_check(0, stream())
        assert e.value.kind == DISPATCH
        backend.stream_check(0, stream())  # reported once
        gone = torch.ones(c.rows, dtype=torch.bool)
        gone[rows] = False
        assert (c.out[gone.cuda()] == 0).all()
        whole = c.out
        c.lens, c.starts = kept, np.cumsum([0] + [n for n, _ in kept]).tolist()
        c.q, c.table = c.q[torch.tensor(rows, device="cuda")], c.table[torch.tensor([i for i, (n, k) in enumerate(lens) if k], device="cuda")]
        check(c, whole[torch.tensor(rows, device="cuda")])


@pytest.mark.parametrize("page", [16, 5])
def test_pages_that_are_not_there_count_as_zeros(backend, page):  # noqa: F811
    for lens in ([(1, 100), (1, 200), (1, 60)], [(1, 100), (2, 200), (1, 60)]):
        c = Cache4(lens, 8, 2, 64, "bf16", page).fill().install(backend)
        c.table[1, 3], c.table[1, 5] = c.n_pages, -1
        forward(backend, c)
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            backend.stream_check(0, stream())
        assert e.value.kind == DISPATCH
        c.table[1, 3] = c.table[1, 5] = 0  # any page: its tokens are zeros for the check
        held, places = c.held, c.places
        missing = torch.cat([torch.arange(3 * page, 4 * page), torch.arange(5 * page, 6 * page)]).cuda()

        def zeroed(keys, at):
            x = held(keys, at)
            if at[0].numel() == 200:
                x[missing] = 0.0
            return x
        c.held = zeroed
        check(c)


def test_length_beyond_the_table(backend):  # noqa: F811
    for lens in ([(1, 100), (1, 30), (1, 60)], [(3, 100), (40, 50), (1, 60)]):
        c = Cache4(lens, 8, 2, 64).fill().install(backend)
        good = forward(backend, c).clone()
        for wrong in (0x7FFFFFFF, -1, c.table.shape[1] * 16 + 1):
            c.kv_len[1] = wrong
            c.out.fill_(7.0)
            forward(backend, c)
            with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
                backend.stream_check(0, stream())
            assert e.value.kind == DISPATCH
            a, b = c.starts[1], c.starts[2]
            assert torch.equal(c.out[:a], good[:a]) and torch.equal(c.out[b:], good[b:]) and (c.out[a:b] == 0).all()


def test_groups_that_are_not_finite_stay_in_their_sequence_and_head(backend):  # noqa: F811
    for lens in ([(1, 100), (1, 300), (1, 60)], [(1, 100), (2, 300), (1, 60)]):
        c = Cache4(lens, 8, 2, 64).fill().install(backend)
        good = forward(backend, c).clone()
        a, b = c.starts[1], c.starts[2]
        places = c.places(1)
        for keys, token in ((False, 250), (True, 20)):
            pairs = c.parts(keys)[1]
            pairs[places[0][token], 1, places[1][token], 1, 1] = math.nan
            forward(backend, c)
            out, was = c.out.view(-1, 8, 64), good.view(-1, 8, 64)
            assert torch.isnan(out[a:b, 4:, 32:]).all()
            assert torch.equal(out[:a], was[:a]) and torch.equal(out[b:], was[b:]) and torch.equal(out[a:b, :4], was[a:b, :4])


@pytest.mark.parametrize("lens", [[(1, 40), (1, 3), (1, 9000)], [(40, 40), (300, 700), (2, 3), (5, 6000)]])
def test_sinks_of_minus_infinity_and_large_ones(backend, lens):  # noqa: F811
    sinks = np.array([-math.inf, 0, 30, -30, 80, -math.inf, 5, -5], dtype=np.float32)
    c = Cache4(lens, 8, 2, 128, "bf16", 16).fill().install(backend, sinks=sinks)
    forward(backend, c)
    check(c)


def test_offsets_beyond_32_bits(backend):  # noqa: F811
    page, d, hk = 16, 128, 2
    block = mer_b200.kv4_block_bytes(d, page)
    far = 5 * (1 << 30)
    pool = torch.zeros(far + 4 * block, dtype=torch.uint8, device="cuda")
    for lens in ([(1, 32)], [(20, 32)]):
        c = Cache4(lens, 4, hk, d, "bf16", page)
        c.n_pages, c.table = 2, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
        c.k, c.v = (torch.as_strided(pool, (2, hk, block), (far, block, 1), i * 2 * block) for i in range(2))
        c.fill().install(backend)
        forward(backend, c)
        check(c)


def test_layers_step_by_step(backend):  # noqa: F811
    # prompts, then tokens one by one; every step appended, attended to and read back
    for group, d in ((32, 128), (64, 80)):
        lens = [33, 100, 7]
        extra = Cache4([(60, 60), (130, 130), (30, 30)], 8, 2, d, "bf16", 16, group)  # a table with room for what comes
        for step in range(12):
            extra.lens = [(n, n) for n in lens] if step == 0 else [(1 + (step % 3 == i) * 2, n) for i, n in enumerate(lens)]
            starts = np.cumsum([0] + [n for n, _ in extra.lens]).tolist()
            extra.starts, extra.rows = starts, starts[-1]
            extra.row_start, extra.kv_len = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, [k for _, k in extra.lens]))
            extra.out = torch.full((starts[-1], 8 * d), 7.0, dtype=extra.kind, device="cuda")
            exact = append(backend, extra, "bf16", rope_dims=d // 2 // 8 * 8)
            extra.q_all = extra.out.clone()
            extra.q = extra.q_all
            backend.attention_forward_device(0, extra.batch(), extra.q.data_ptr(), extra.out.data_ptr(), stream())
            k, v = read(backend, extra)
            backend.stream_check(0, stream())
            for got, a in ((k, 8), (v, 10)):
                codes, scales, minima = quantised(exact[:, a:a + 2], group)
                assert torch.equal(got.view(-1, 2, d), numbers(codes, scales, minima, group).float())
            check(extra)
            lens = [n + m for n, m in zip(lens, [1 + ((step + 1) % 3 == i) * 2 for i in range(3)])]


def test_captured_call_follows_its_tables(backend):  # noqa: F811
    for behind in (0, 6):  # single tokens, and any rows
        c = Cache4([(1, 400), (1, 60), (1, 200)], 8, 2, 128, "bf16", 16, behind=behind).fill().install(backend)
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            backend.attention_forward_device(0, c.batch(), c.q.data_ptr(), c.out.data_ptr(), side.cuda_stream)
        for lens in ([(1, 400), (1, 60), (1, 200)], [(1, 16), (0, 60), (1, 177)], *([[(5, 333), (1, 1), (3, 64)]] if behind else [])):
            c.lens, c.starts = lens, np.cumsum([0] + [n for n, _ in lens]).tolist()
            c.row_start.copy_(torch.tensor(c.starts, dtype=torch.int32))
            c.kv_len.copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))
            c.out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            check(c)


def test_beside_a_cache_of_16_bits(backend):  # noqa: F811
    # layers of both kinds share the backend's workspace, one call behind the other
    from test_gpu_attention import Cache
    for lens in (LENS["decode"], LENS["draft"]):
        a = Cache(lens, 8, 2, 128, "bf16", 16).fill().install(backend, layer=1)
        c = Cache4(lens, 8, 2, 128, "bf16", 16).fill().install(backend)
        for _ in range(3):
            a.forward(backend, layer=1)
            forward(backend, c)
        backend.stream_check(0, stream())
        a.check()
        check(c)


def test_other_stream(backend):  # noqa: F811
    c = Cache4(LENS["decode"], 8, 2, 128, "bf16", 16).fill().install(backend)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward(backend, c)
        backend.stream_check(0, side.cuda_stream)
    check(c)
