"""Attention over a paged cache (mer_attention_install, mer_kv_append_device, mer_attention_forward_device) against the formulas in
64 bits.

Bounds.  A rounding to a type is off by at most u = eps / 2 of the value.  Appended values: fp32 arithmetic on a head (about a
dozen operations, 2^-24 each, relative to the head's largest value: 2^-19 covers them) and one rounding.  Attention: the weights of the
second product are rounded to the cache's type, so u * A with A = sum_j p_j |v_j|; the output is, u * |o|; a score's fp32 sum of D products is
off by at most (D + 3) 2^-24 * scale * sum |q k|, which moves a weight, and the sum it is divided by, by as much in proportion; exponentials,
sums and joins add less than 2^-18."""
import math

import numpy as np
import pytest

import mer_b200

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, mer_b200.VALUE_F32), "f16": (torch.float16, mer_b200.VALUE_F16), "bf16": (torch.bfloat16, mer_b200.VALUE_BF16)}
INVALID, DISPATCH = mer_b200.GpuExpertDispatchErrorKind.InvalidArgument, mer_b200.GpuExpertDispatchErrorKind.ValidationDispatch


@pytest.fixture(scope="module")
def backend():
    with mer_b200.Backend(mer_b200.DTYPE_Q8_0, 64, 64, 1 << 20, 1, max_tokens=1, max_top_k=1) as b:
        yield b


class Cache:
    """Sequences of (new rows, tokens with them) in a pool of pages; everything that no sequence holds is NaN."""

    def __init__(self, lens, q_heads, kv_heads, d, kind="bf16", page=16, heads_first=False, seed=0, behind=0, wide=0, q_gap=0):
        g = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.hq, self.hk, self.d, self.page = lens, q_heads, kv_heads, d, page
        self.kind, self.value_type = TYPES[kind]
        held = [-(-k // page) for _, k in lens]
        self.n_pages, widest = sum(held) + 2, max(held + [1]) + wide
        shape = (self.n_pages, kv_heads, page, d) if heads_first else (self.n_pages, page, kv_heads, d)
        self.k_pool, self.v_pool = (torch.full(shape, math.nan, dtype=self.kind, device="cuda") for _ in range(2))
        self.k, self.v = (p.transpose(1, 2) if heads_first else p for p in (self.k_pool, self.v_pool))
        order = torch.randperm(self.n_pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(lens), widest), -1, dtype=torch.int32, device="cuda")
        at, starts = 0, [0]
        for i, (n, k) in enumerate(lens):
            self.table[i, :held[i]] = order[at:at + held[i]]
            at += held[i]
            starts.append(starts[-1] + n)
        self.starts, self.rows = starts, starts[-1] + behind
        self.row_start, self.kv_len = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, [k for _, k in lens]))
        self.q_all = torch.randn((max(1, self.rows), q_heads * d + q_gap), device="cuda", generator=g).to(self.kind)
        self.q = self.q_all[:, :q_heads * d]
        self.out = torch.full((max(1, self.rows), q_heads * d), 7.0, dtype=self.kind, device="cuda")

    def places(self, i, first=0, last=None):
        at = torch.arange(first, self.lens[i][1] if last is None else last, device="cuda")
        return self.table[i, at // self.page].long(), at % self.page

    def fill(self, first=None):
        """Tokens of every sequence (from first[i] on)."""
        for i, (_, k) in enumerate(self.lens):
            lo = 0 if first is None else first[i]
            if k > lo:
                for x in (self.k, self.v):
                    x[self.places(i, lo)] = torch.randn((k - lo, self.hk, self.d), device="cuda", generator=self.gen).to(self.kind)
        return self

    def batch(self, **kw):
        f = dict(k_pages=self.k.data_ptr(), v_pages=self.v.data_ptr(), n_pages=self.n_pages, page_stride=self.k.stride(0), token_stride=self.k.stride(1),
                 head_stride=self.k.stride(2), page_table=self.table.data_ptr(), table_stride=self.table.shape[1], row_start=self.row_start.data_ptr(),
                 kv_len=self.kv_len.data_ptr(), n_seqs=len(self.lens), n_rows=self.rows)
        return mer_b200.KvBatch(**{**f, **kw})

    def install(self, b, layer=0, **kw):
        b.install_attention(layer, self.hq, self.hk, self.d, self.value_type, self.page, **kw)
        self.opts = kw
        return self

    def forward(self, b, layer=0, **kw):
        b.attention_forward_device(layer, self.batch(**kw), self.q.data_ptr(), self.out.data_ptr(), torch.cuda.current_stream().cuda_stream,
                                   q_stride=self.q_all.stride(0))
        return self.out

    def check(self, out=None):
        out = self.out if out is None else out
        u, window, g = torch.finfo(self.kind).eps / 2, self.opts.get("window", 0), self.hq // self.hk
        scale = self.opts.get("scale", 0) or self.d ** -0.5
        sinks = self.opts.get("sinks")
        for i, (n, k) in enumerate(self.lens):
            if n == 0 or k == 0:
                continue
            pos = torch.arange(k - n, k, device="cuda")
            lo = max(0, k - n - window + 1) if window else 0  # what is before it may be anything
            at = torch.arange(lo, k, device="cuda")
            keys, values = (x[self.places(i, lo)].double().transpose(0, 1) for x in (self.k, self.v))
            q = self.q[self.starts[i]:self.starts[i + 1]].double().view(n, self.hk, g, self.d).permute(1, 2, 0, 3)
            s = torch.einsum("hgnd,htd->hgnt", q, keys) * scale
            size = torch.einsum("hgnd,htd->hgnt", q.abs(), keys.abs()) * scale
            hidden = at > pos[:, None]
            if window:
                hidden |= at <= pos[:, None] - window
            s = s.masked_fill(hidden, -math.inf)
            total = torch.logsumexp(s, 3, keepdim=True)
            if sinks is not None:
                total = torch.logaddexp(total, torch.tensor(sinks, dtype=torch.float64, device="cuda").view(self.hk, g, 1, 1))
            p = (s - total).exp()
            p = torch.where(hidden.all(1)[:, None], torch.zeros_like(p), p)
            want = torch.einsum("hgnt,htd->hgnd", p, values)
            a = torch.einsum("hgnt,htd->hgnd", p, values.abs())
            # only what a row sees moves its weights
            move = torch.where(hidden, torch.zeros_like(size), size).amax(3, keepdim=True) * (self.d + 3) * 2.0 ** -24
            bound = u * (a + want.abs()) * 1.01 + (2 * move + 2.0 ** -18) * a + 2.0 ** -24
            got = out[self.starts[i]:self.starts[i + 1]].double().view(n, self.hk, g, self.d).permute(1, 2, 0, 3)
            worst = ((got - want).abs() / bound).max().item()
            assert worst <= 1.0, (i, n, k, worst)
        assert (out[self.starts[-1]:] == 7.0).all()


LENS = {
    "one": [(1, 1)],
    "decode": [(1, 77), (1, 1), (1, 300), (1, 16), (1, 129)],
    "long": [(1, 9000)],
    "idle": [(0, 40), (1, 33), (0, 0), (0, 5), (1, 90), (0, 7)],
    "draft": [(5, 70), (3, 3), (7, 513), (2, 1025)],
    "prompts": [(33, 33), (100, 257), (1, 50), (200, 200)],
    "chunk": [(300, 1500)],
}


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("q_heads,kv_heads,d,kind,page", [(8, 1, 128, "bf16", 16), (32, 4, 128, "f16", 32), (6, 6, 64, "bf16", 1), (20, 4, 80, "f16", 24),
                                                          (2, 1, 8, "bf16", 3), (40, 1, 64, "f16", 64), (4, 2, 256, "bf16", 16), (7, 1, 136, "f16", 5),
                                                          (2, 2, 8, "f16", 32), (3, 1, 24, "bf16", 16), (300, 1, 8, "f16", 16), (130, 1, 200, "bf16", 128), (1, 1, 256, "f16", 24)])
def test_attention(backend, lens, q_heads, kv_heads, d, kind, page):
    c = Cache(LENS[lens], q_heads, kv_heads, d, kind, page, behind=3).fill().install(backend)
    c.forward(backend)
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    c.check()


@pytest.mark.parametrize("lens", ["decode", "draft", "prompts", "chunk", "long"])
@pytest.mark.parametrize("window", [1, 2, 17, 128, 1000])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_window_and_sinks(backend, lens, window, d):
    # tokens before every window are NaN, and so are the pages that hold only such tokens
    c = Cache(LENS[lens], 8, 2, d, "bf16", 16, heads_first=True, seed=window)
    c.fill([max(0, k - n - window + 1) for n, k in c.lens])
    c.install(backend, window=window, sinks=np.linspace(-3, 4, 8).astype(np.float32), scale=0.2)
    c.forward(backend)
    c.check()


def test_many_sequences(backend):
    rng = np.random.default_rng(5)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 4, 700), rng.integers(0, 200, 700))]
    c = Cache(lens, 8, 2, 64, "f16", 8, seed=2, behind=5).fill().install(backend)
    c.forward(backend)
    c.check()


def test_large_scores_and_small_weights(backend):
    # one key far above thousands of equal ones: what these sum to counts
    c = Cache([(1, 6000)], 4, 1, 64, "f16", 16).fill().install(backend)
    c.q.mul_(0).add_(1.0)
    at = c.places(0)
    c.k[at] = 0.0
    c.k[at[0][3], at[1][3]] = 10.0 * 8 / 64
    c.forward(backend)
    c.check()
    c.q.mul_(300.0)  # scores of thousands
    c.forward(backend)
    c.check()


def test_query_and_output_strides(backend):
    c = Cache(LENS["draft"], 8, 2, 64, "bf16", 16, q_gap=64).fill().install(backend)
    wide = torch.full((c.rows, 8 * 64 + 24), 3.0, dtype=c.kind, device="cuda")
    backend.attention_forward_device(0, c.batch(), c.q.data_ptr(), wide.data_ptr(), torch.cuda.current_stream().cuda_stream, c.q_all.stride(0), wide.stride(0))
    c.check(wide[:, :512])
    assert (wide[:, 512:] == 3.0).all()


@pytest.mark.parametrize("gap", [8, 64, 256])
def test_query_rows_that_have_no_map(backend, gap):
    # rows that are no whole number of heads apart are copied one by one
    for d in (64, 256):
        c = Cache(LENS["prompts"], 8, 2, d, "f16", 16, q_gap=gap, behind=2).fill().install(backend)
        c.forward(backend)
        c.check()


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (2, 0, 1), (1, 0, 2), (2, 1, 0)])
@pytest.mark.parametrize("lens", ["decode", "prompts"])
def test_pages_tokens_and_heads_in_any_order(backend, order, lens):
    # the pool's dimensions [page, token, head] outermost first, with a hole behind each token's head
    c = Cache(LENS[lens], 8, 4, 64, "bf16", 16)
    sizes = [(c.n_pages, 16, 4)[o] for o in order]
    for name in ("k", "v"):
        pool = torch.full((*sizes, 72), math.nan, dtype=c.kind, device="cuda")
        setattr(c, name, pool.permute(*(order.index(i) for i in range(3)), 3)[..., :64])
    c.fill().install(backend)
    c.forward(backend)
    c.check()
    append_and_check(backend, c, "bf16", norm=True, rope_dims=64, pairs=False)


def test_keys_and_values_of_one_pool(backend):
    # [page][keys, values][token][head]
    for lens in ("decode", "chunk"):
        c = Cache(LENS[lens], 8, 4, 128, "f16", 32)
        pool = torch.full((c.n_pages, 2, 32, 4, 128), math.nan, dtype=c.kind, device="cuda")
        c.k, c.v = pool[:, 0], pool[:, 1]
        c.fill().install(backend)
        c.forward(backend)
        c.check()


def test_same_bits_every_time(backend):
    c = Cache([(1, 5000), (3, 900), (40, 2000), (1, 2)], 16, 2, 128, "bf16", 16).fill().install(backend)
    first = c.forward(backend).clone()
    for _ in range(20):
        assert torch.equal(c.forward(backend), first)


def test_sequence_with_more_rows_than_tokens(backend):
    c = Cache([(2, 50), (6, 4), (3, 0), (1, 20)], 8, 2, 64).fill().install(backend)
    c.forward(backend)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    assert e.value.kind == DISPATCH
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)  # reported once
    assert (c.out[2:4] == 0).all() and (c.out[8:11] == 0).all()
    whole = c.out
    c.lens, c.starts = [(2, 50), (4, 4), (1, 20)], [0, 2, 6, 7]
    rows = torch.tensor([0, 1, 4, 5, 6, 7, 11], device="cuda")
    c.q, c.table = c.q[rows], c.table[torch.tensor([0, 1, 3], device="cuda")]
    c.check(whole[rows])


@pytest.mark.parametrize("wrong", ["number", "table"])
def test_page_that_is_not_there(backend, wrong):
    c = Cache([(1, 100), (2, 200), (1, 60)], 8, 2, 64).fill().install(backend)
    good = c.forward(backend).clone()
    if wrong == "number":
        c.table[1, 3] = c.n_pages
        c.table[1, 5] = -1
        c.forward(backend)
    else:
        c.forward(backend, table_stride=c.table.shape[1])
        narrow = c.table[:, :7].contiguous()  # 112 tokens: sequence 1 has more
        c.forward(backend, page_table=narrow.data_ptr(), table_stride=7)
    with pytest.raises(mer_b200.GpuExpertDispatchError):
        backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(c.out[0], good[0]) and torch.equal(c.out[3], good[3])
    assert torch.isfinite(c.out.float()).all()


def test_length_beyond_the_table(backend):
    # lengths that were never written: nothing of such a sequence is run, the others are
    for lens in ([(1, 100), (1, 30), (1, 60)], [(3, 100), (40, 50), (1, 60)]):
        c = Cache(lens, 8, 2, 64).fill().install(backend)
        good = c.forward(backend).clone()
        for wrong in (0x7FFFFFFF, -1, c.table.shape[1] * 16 + 1):
            c.kv_len[1] = wrong
            c.out.fill_(7.0)
            c.forward(backend)
            with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
                backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
            assert e.value.kind == DISPATCH
            a, b = c.starts[1], c.starts[2]
            assert torch.equal(c.out[:a], good[:a]) and torch.equal(c.out[b:], good[b:]) and (c.out[a:b] == 0).all()
            before = c.k_pool.view(torch.int16).clone()
            x = torch.randn((c.rows, 512), device="cuda", dtype=c.kind)
            rows = mer_b200.QkvRows(k=x.data_ptr(), v=x.data_ptr(), k_stride=512, v_stride=512, value_type=c.value_type)
            c.row_start.copy_(torch.tensor([0, 0, b - a, b - a], dtype=torch.int32))  # that sequence alone
            backend.kv_append_device(0, c.batch(n_rows=b - a), rows, torch.cuda.current_stream().cuda_stream)
            with pytest.raises(mer_b200.GpuExpertDispatchError):
                backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
            assert torch.equal(c.k_pool.view(torch.int16), before)
            c.row_start.copy_(torch.tensor(c.starts, dtype=torch.int32))


def test_values_that_are_not_finite_stay_in_their_sequence(backend):
    c = Cache([(1, 100), (2, 300), (1, 60)], 8, 2, 64).fill().install(backend)
    good = c.forward(backend).clone()
    pages, slots = c.places(1)
    c.v[pages[250], slots[250], 1, 5] = math.nan
    c.forward(backend)
    out = c.out.view(-1, 8, 64)
    assert torch.isnan(out[1:3, 4:, 5]).all()
    out[1:3, 4:, 5] = good.view(-1, 8, 64)[1:3, 4:, 5]
    assert torch.equal(c.out, good)
    c.k[pages[20], slots[20], 0, 3] = math.nan
    c.forward(backend)
    assert torch.isnan(out[1:3, :4]).all() and torch.equal(out[0], good.view(-1, 8, 64)[0])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 40), (1, 3), (1, 2000)], [(40, 40), (300, 700), (2, 3), (3, 3)]])
def test_scores_of_minus_infinity_have_no_weight(backend, lens, d):
    c = Cache(lens, 8, 2, d, "bf16", 16).fill().install(backend)
    c.q.view(-1, 8, d)[:, :, 0] = c.q.view(-1, 8, d)[:, :, 0].abs() + 0.5  # -infinity times it, plus what is finite
    for i, (n, k) in enumerate(lens):
        pages, slots = c.places(i, 0, 3)
        c.k[pages, slots, 0, 0] = -math.inf  # the first three tokens, for the first key head
    c.forward(backend)
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    u = torch.finfo(c.kind).eps / 2
    for i, (n, k) in enumerate(lens):
        keys, values = (x[c.places(i)].double().transpose(0, 1) for x in (c.k, c.v))
        q = c.q[c.starts[i]:c.starts[i + 1]].double().view(n, 2, 4, d).permute(1, 2, 0, 3)
        s = torch.einsum("hgnd,htd->hgnt", q, keys) * d ** -0.5
        hidden = torch.arange(k, device="cuda") > torch.arange(k - n, k, device="cuda")[:, None]
        s = s.masked_fill(hidden, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, 3), nan=0.0)
        want, a = torch.einsum("hgnt,htd->hgnd", p, values), torch.einsum("hgnt,htd->hgnd", p, values.abs())
        # |q| |k| scale is below d * 5 * 5 / sqrt(d) here
        bound = u * (a + want.abs()) * 1.01 + (2 * 25 * d ** 0.5 * (d + 3) * 2.0 ** -24 + 2.0 ** -18) * a + 2.0 ** -24
        got = c.out[c.starts[i]:c.starts[i + 1]].double().view(n, 2, 4, d).permute(1, 2, 0, 3)
        assert ((got - want).abs() <= bound).all(), (i, n, k)


# ------------------------------------------------------------------------------------------------ appending


def append_and_check(b, c, source, *, norm, rope_dims, pairs, theta=1e4, rope_scale=1.0, gap=0, offset=0, with_q=True, layer=0, in_place=False):
    dtype, value_type = TYPES[source]
    hq, hk, d = c.hq, c.hk, c.d
    width = (hq + 2 * hk) * d
    store = torch.randn(c.rows * (width + gap) + offset, device="cuda", generator=c.gen).mul_(2).to(dtype)
    x = store[offset:].view(c.rows, width + gap)
    rng = np.random.default_rng(9)
    qw, kw = ((1 + 0.3 * rng.standard_normal(d)).astype(np.float32) for _ in range(2))
    freq = theta ** (-np.arange(rope_dims // 2) / max(1, rope_dims // 2))
    c.install(b, layer, q_norm=qw if norm else None, k_norm=kw if norm else None, norm_eps=1e-5, rope_freq=freq if rope_dims else None, rope_pairs=pairs,
              rope_scale=rope_scale)
    exact = x[:, :width].double().view(c.rows, hq + 2 * hk, d)
    gain = np.ones((hq + 2 * hk, d))
    if norm:
        gain[:hq], gain[hq:hq + hk] = qw, kw
        size = (exact.square().mean(2, keepdim=True) + 1e-5).sqrt()
        size[:, hq + hk:] = 1.0
        exact = exact / size * torch.tensor(gain, device="cuda")
    pos = torch.full((c.rows,), -1.0, dtype=torch.float64, device="cuda")
    for i, (n, k) in enumerate(c.lens):
        pos[c.starts[i]:c.starts[i + 1]] = torch.arange(k - n, k, device="cuda", dtype=torch.float64)
    if rope_dims:
        angle = pos[:, None, None] * torch.tensor(freq, device="cuda")
        r = rope_dims
        one, two = (slice(0, r, 2), slice(1, r, 2)) if pairs else (slice(0, r // 2), slice(r // 2, r))
        turned = exact.clone()
        a, z = exact[:, :hq + hk, one], exact[:, :hq + hk, two]
        turned[:, :hq + hk, one] = (a * angle.cos() - z * angle.sin()) * rope_scale
        turned[:, :hq + hk, two] = (a * angle.sin() + z * angle.cos()) * rope_scale
        exact = turned
    e = x.element_size()
    k_want, v_want = c.k.clone(), c.v.clone()
    q_out = x[:, :hq * d] if in_place else c.out
    q_before = q_out.clone()
    rows = mer_b200.QkvRows(q=x.data_ptr() if with_q else None, k=x.data_ptr() + e * hq * d, v=x.data_ptr() + e * (hq + hk) * d,
                            q_out=q_out.data_ptr() if with_q else None, q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0),
                            q_out_stride=q_out.stride(0), value_type=value_type)
    b.kv_append_device(layer, c.batch(), rows, torch.cuda.current_stream().cuda_stream)
    u = torch.finfo(c.kind).eps / 2

    def near(got, want):
        bound = u * want.abs() * 1.0001 + 2.0 ** -19 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25
        worst = ((got.double() - want).abs() / bound).max().item() if want.numel() else 0.0
        assert worst <= 1.0, worst

    placed = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
    for i, (n, k) in enumerate(c.lens):
        lo = max(0, k - n)
        skip = max(0, n - k)
        sl = slice(c.starts[i] + skip, c.starts[i + 1])
        placed[sl] = True
        if sl.start < sl.stop:
            pages, slots = c.places(i, lo)
            near(c.k[pages, slots], exact[sl, hq:hq + hk])
            near(c.v[pages, slots], exact[sl, hq + hk:])
            k_want[pages, slots], v_want[pages, slots] = c.k[pages, slots], c.v[pages, slots]
    # nothing else has changed (NaN included)
    as_bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(as_bits(c.k), as_bits(k_want)) and torch.equal(as_bits(c.v), as_bits(v_want))
    if with_q:
        near(q_out[placed].view(-1, hq, d), exact[placed, :hq])
    keep = ~placed if with_q else torch.ones_like(placed)
    assert torch.equal(as_bits(q_out[keep]), as_bits(q_before[keep]))


@pytest.mark.parametrize("source", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,d,kind,page,rope_dims,pairs,norm", [
    (8, 2, 128, "bf16", 16, 128, False, True), (32, 4, 128, "f16", 32, 128, True, True), (5, 1, 80, "bf16", 24, 40, False, True),
    (4, 4, 64, "f16", 1, 32, True, False), (3, 1, 8, "bf16", 5, 6, False, True), (2, 1, 256, "f16", 16, 256, False, True), (2, 2, 136, "bf16", 8, 0, False, True),
    (2, 1, 72, "f16", 16, 70, True, False), (2, 1, 248, "bf16", 7, 30, False, True), (16, 2, 96, "bf16", 64, 96, True, True)])
def test_append(backend, source, q_heads, kv_heads, d, kind, page, rope_dims, pairs, norm):
    c = Cache([(1, 1), (0, 9), (3, 70), (1, 1000), (40, 41)], q_heads, kv_heads, d, kind, page, heads_first=page == 24, behind=2)
    append_and_check(backend, c, source, norm=norm, rope_dims=rope_dims, pairs=pairs, rope_scale=1.25 if pairs else 1.0)


@pytest.mark.parametrize("offset,gap", [(1, 0), (4, 12), (0, 3), (8, 8)])
def test_append_rows_at_odd_places(backend, offset, gap):
    c = Cache([(5, 9), (1, 40)], 8, 2, 64, "f16", 16)
    for source in ("f32", "bf16"):
        append_and_check(backend, c, source, norm=True, rope_dims=64, pairs=False, gap=gap, offset=offset)


def test_append_many_rows(backend):
    c = Cache([(1500, 1700), (0, 3), (2500, 2500), (1, 4)], 8, 2, 128, "bf16", 16, behind=7)
    append_and_check(backend, c, "bf16", norm=True, rope_dims=128, pairs=False)
    append_and_check(backend, c, "f32", norm=False, rope_dims=64, pairs=True)


def test_append_thousands_of_sequences(backend):
    rng = np.random.default_rng(6)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 3, 3000), rng.integers(0, 20, 3000))]
    c = Cache(lens, 2, 1, 64, "f16", 8, behind=3)
    x = torch.randn((c.rows, 256), device="cuda").to(c.kind)
    c.install(backend)
    rows = mer_b200.QkvRows(k=x.data_ptr() + 256, v=x.data_ptr() + 384, k_stride=256, v_stride=256, value_type=c.value_type)
    backend.kv_append_device(0, c.batch(), rows, torch.cuda.current_stream().cuda_stream)
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    seq = torch.tensor([i for i, (n, _) in enumerate(lens) for _ in range(n)], device="cuda")
    pos = torch.tensor([k - n + j for n, k in lens for j in range(n)], device="cuda")
    pages = c.table[seq, pos // 8].long()
    assert torch.equal(c.k[pages, pos % 8, 0], x[:len(seq), 128:192]) and torch.equal(c.v[pages, pos % 8, 0], x[:len(seq), 192:])
    assert int((~torch.isnan(c.k_pool)).sum()) == 64 * len(seq)


def test_append_far_positions(backend):
    # positions of a million: an angle in 32 bits would be off by 0.06
    c = Cache([(2, 1 << 20), (1, 999999)], 2, 1, 64, "f16", 1 << 14)
    append_and_check(backend, c, "f32", norm=False, rope_dims=64, pairs=False, theta=1.5)


def test_append_without_queries_and_in_place(backend):
    c = Cache([(3, 8), (1, 40)], 8, 2, 64, "bf16", 16)
    append_and_check(backend, c, "bf16", norm=True, rope_dims=64, pairs=False, with_q=False)
    append_and_check(backend, c, "bf16", norm=True, rope_dims=64, pairs=False, in_place=True)


def test_append_rows_without_a_place(backend):
    c = Cache([(5, 2), (2, 20), (1, 0)], 4, 2, 64, "bf16", 16)
    append_and_check(backend, c, "bf16", norm=True, rope_dims=64, pairs=False)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    assert e.value.kind == DISPATCH
    # pages that are not there: nothing is written
    c.table[1, 1] = c.n_pages + 5
    before = c.k_pool.clone()
    x = torch.randn((c.rows, 8 * 64), device="cuda", dtype=c.kind)
    rows = mer_b200.QkvRows(k=x.data_ptr(), v=x.data_ptr(), k_stride=512, v_stride=512, value_type=c.value_type)
    backend.kv_append_device(0, c.batch(), rows, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(mer_b200.GpuExpertDispatchError):
        backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    changed = (c.k_pool.view(torch.int16) != before.view(torch.int16)).flatten(1).any(1)
    assert set(torch.nonzero(changed).flatten().tolist()) <= {int(c.table[0, 0])}


def test_offsets_beyond_32_bits(backend):
    # two pages whose values lie more than 2^31 values apart
    c = Cache([(4, 30)], 4, 1, 64, "bf16", 16)
    far = (1 << 31) + 4096
    try:
        pool = torch.zeros(2 * far + 64 * 16 * 2, dtype=c.kind, device="cuda")
    except torch.OutOfMemoryError:
        pytest.skip("no room for a cache of 8 GB")
    half = far + 16 * 64
    c.k, c.v = (torch.as_strided(pool, (2, 16, 1, 64), (far, 64, 64, 1), o) for o in (0, half))
    c.n_pages = 2
    c.table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    c.fill()
    append_and_check(backend, c, "f32", norm=True, rope_dims=64, pairs=False)
    c.q_all = c.q = torch.randn((4, 256), device="cuda", generator=c.gen).to(c.kind)
    c.forward(backend)
    c.check()


# ------------------------------------------------------------------------------------------------ as they are used


def test_layers_step_by_step(backend):
    """A prompt in two chunks and then tokens one by one, through two layers' caches, equal the whole prompt at once."""
    hq, hk, d, total = 8, 2, 64, 40
    gen = torch.Generator(device="cuda").manual_seed(3)
    freq = 1e4 ** (-np.arange(32) / 32)
    qkv = [torch.randn((total, (hq + 2 * hk) * d), device="cuda", generator=gen) for _ in range(2)]
    stream = torch.cuda.current_stream().cuda_stream
    outs = {}
    for name, steps in (("whole", [40]), ("steps", [13, 20, 1, 1, 1, 4])):
        for layer in range(2):
            c = Cache([(total, total)], hq, hk, d, "bf16", 8, seed=layer)
            c.install(backend, layer, q_norm=np.ones(d, np.float32), rope_freq=freq, window=0 if layer else 11)
            done, got = 0, []
            for n in steps:
                c.row_start.copy_(torch.tensor([0, n], dtype=torch.int32))
                c.kv_len.fill_(done + n)
                x = qkv[layer][done:done + n]
                rows = mer_b200.QkvRows(q=x.data_ptr(), k=x.data_ptr() + 4 * hq * d, v=x.data_ptr() + 4 * (hq + hk) * d, q_out=c.q.data_ptr(),
                                        q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0), value_type=mer_b200.VALUE_F32)
                backend.kv_append_device(layer, c.batch(n_rows=n), rows, stream)
                backend.attention_forward_device(layer, c.batch(n_rows=n), c.q.data_ptr(), c.out.data_ptr(), stream)
                got.append(c.out[:n].clone())
                done += n
            outs[name, layer] = torch.cat(got)
            if name == "whole":
                c.check()
            else:
                # the same keys, values and queries; weights rounded in another order of blocks: as far apart as two checks allow
                a, z = outs["whole", layer].double(), outs["steps", layer].double()
                assert (a - z).abs().max() <= 4 * torch.finfo(torch.bfloat16).eps * a.abs().max()
    backend.stream_check(0, stream)


def test_beside_the_expert_layers_of_one_backend():
    """The calls of two decoder layers on one stream, nothing waited for between them: rows appended, attended to, and through the experts."""
    synth = __import__("importlib").import_module("mer_b200.synth")
    dtype, experts, d_model, d_ff, layers, n = mer_b200.DTYPE_Q8_0, 4, 256, 256, 2, 6
    stride = (256 + mer_b200.expert_bytes(dtype, d_model, d_ff) + 4095) // 4096 * 4096
    with mer_b200.Backend(dtype, d_model, d_ff, stride * experts * layers, experts * layers, max_tokens=64, max_top_k=2) as b:
        for e in range(experts * layers):
            b.admit(e, 1, synth.make_expert_blob(dtype, d_model, d_ff, 1, e // experts, e % experts))
        for layer in range(layers):
            mer_b200.LinearGate(synth.make_router(experts, d_model, layer), experts, d_model, 2).bind(b, layer)
        stream = torch.cuda.current_stream().cuda_stream
        for lens in ([(1, 40), (1, 700), (1, 3), (1, 90), (1, 16), (1, 17)], [(6, 300)]):
            caches = [Cache(lens, 8, 2, 64, "bf16", 16, seed=l).fill() for l in range(layers)]
            x = torch.randn((n, d_model), device="cuda")
            qkv = torch.randn((n, 12 * 64), device="cuda")
            rows = lambda c: mer_b200.QkvRows(q=qkv.data_ptr(), k=qkv.data_ptr() + 4 * 512, v=qkv.data_ptr() + 4 * 640, q_out=c.q.data_ptr(), q_stride=768,  # noqa: E731
                                              k_stride=768, v_stride=768, value_type=mer_b200.VALUE_F32)
            for layer, c in enumerate(caches):
                c.install(b, layer, rope_freq=1e4 ** (-np.arange(32) / 32))
            outs = [[], []]
            for wait in (True, False):  # call by call, then all at once, several times
                for _ in range(1 if wait else 8):
                    y = [x.clone() for _ in range(layers + 1)]
                    for layer, c in enumerate(caches):
                        b.kv_append_device(layer, c.batch(), rows(c), stream)
                        if wait:
                            torch.cuda.synchronize()
                        b.attention_forward_device(layer, c.batch(), c.q.data_ptr(), c.out.data_ptr(), stream)
                        if wait:
                            torch.cuda.synchronize()
                        b.moe_layer_forward_device(layer, y[layer].data_ptr(), n, y[layer + 1].data_ptr(), stream)
                        if wait:
                            torch.cuda.synchronize()
                    torch.cuda.synchronize()
                    outs[not wait].append([y[-1].clone(), *(c.out.clone() for c in caches)])
            for got in outs[1]:
                assert all(torch.equal(a, w) for a, w in zip(got, outs[0][0]))
            for c in caches:
                c.check()
        b.stream_check(0, stream)


def test_captured_call_follows_its_tables(backend):
    """One graph for every step of a batch: lengths, tables and rows change between replays, sequences come and go."""
    hq, hk, d = 8, 2, 64
    c = Cache([(1, 200), (1, 200), (1, 200), (1, 200)], hq, hk, d, "bf16", 16).fill()
    c.install(backend, 0, rope_freq=1e4 ** (-np.arange(32) / 32))
    x = torch.randn((4, (hq + 2 * hk) * d), device="cuda", dtype=torch.bfloat16)
    rows = mer_b200.QkvRows(q=x.data_ptr(), k=x.data_ptr() + 2 * hq * d, v=x.data_ptr() + 2 * (hq + hk) * d, q_out=c.q.data_ptr(), q_stride=x.stride(0),
                            k_stride=x.stride(0), v_stride=x.stride(0), value_type=mer_b200.VALUE_BF16)
    batch = c.batch()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        s = torch.cuda.current_stream().cuda_stream
        backend.kv_append_device(0, batch, rows, s)
        backend.attention_forward_device(0, batch, c.q.data_ptr(), c.out.data_ptr(), s)
    check_steps = [[(1, 5), (1, 190), (1, 64), (1, 1)], [(1, 6), (0, 190), (2, 66), (1, 2)], [(0, 6), (0, 190), (0, 66), (4, 4)], [(0, 0)] * 4]
    for step, lens in enumerate(check_steps):
        c.lens, c.starts = lens, np.concatenate([[0], np.cumsum([n for n, _ in lens])]).tolist()
        c.row_start.copy_(torch.tensor(c.starts, dtype=torch.int32))
        c.kv_len.copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))
        x.copy_(torch.randn(x.shape, device="cuda").to(x.dtype))
        c.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        c.check()
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)


def test_captured_chunks_follow_their_tables(backend):
    # the same for the kernel of many rows: 96 rows at most, in any split, or none
    c = Cache([(1, 400)] * 5, 8, 2, 128, "bf16", 16).fill()
    c.install(backend, 0)
    c.rows = 96
    c.q_all = c.q = torch.randn((96, 1024), device="cuda").to(c.kind)
    c.out = torch.empty_like(c.q)
    batch, side, graph = c.batch(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        backend.attention_forward_device(0, batch, c.q.data_ptr(), c.out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for lens in ([(1, 400), (90, 390), (0, 3), (4, 4), (1, 77)], [(0, 400)] * 5, [(96, 96), (0, 0), (0, 1), (0, 400), (0, 2)], [(1, 300)] * 5, [(0, 5)] * 4 + [(96, 400)]):
        c.lens, c.starts = lens, np.concatenate([[0], np.cumsum([n for n, _ in lens])]).tolist()
        c.row_start.copy_(torch.tensor(c.starts, dtype=torch.int32))
        c.kv_len.copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))
        for _ in range(3):
            c.out.fill_(7.0)
            graph.replay()
        torch.cuda.synchronize()
        c.check()
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)


def test_other_stream_and_two_backends(backend):
    c = Cache([(1, 3000), (1, 700)], 8, 2, 128, "bf16", 16).fill().install(backend)
    want = c.forward(backend).clone()
    torch.cuda.synchronize()
    with mer_b200.Backend(mer_b200.DTYPE_Q8_0, 64, 64, 1 << 20, 1, max_tokens=1, max_top_k=1) as other:
        c.install(other)
        outs = [torch.empty_like(c.out) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(30):  # each backend's calls on a stream of its own, at once
            for b, s, o in zip((backend, other), streams, outs):
                b.attention_forward_device(0, c.batch(), c.q.data_ptr(), o.data_ptr(), s.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_empty_batches_and_layer_installed_anew(backend):
    c = Cache([(1, 30)], 8, 2, 64).fill().install(backend)
    before = backend.snapshot()["kernel_launches"]
    c.forward(backend, n_rows=0)
    c.forward(backend, n_seqs=0)
    assert (c.out == 7.0).all() and backend.snapshot()["kernel_launches"] == before
    c.forward(backend)
    c.check()
    assert backend.snapshot()["kernel_launches"] > before
    c.install(backend, window=4, scale=1.0)
    c.forward(backend)
    c.check()


# ------------------------------------------------------------------------------------------------ refusals


@pytest.mark.parametrize("change", [dict(q_heads=0), dict(kv_heads=0), dict(q_heads=7), dict(head_dim=0), dict(head_dim=12), dict(head_dim=264),
                                    dict(cache_type=mer_b200.VALUE_F32), dict(cache_type=9), dict(page_tokens=0), dict(scale=-1.0), dict(scale=math.nan),
                                    dict(norm_eps=-1.0), dict(rope_scale=math.inf), dict(rope_freq=np.ones(33)), dict(rope_freq=np.array([math.nan]))])
def test_refused_layers(backend, change):
    good = dict(layer=5, q_heads=8, kv_heads=2, head_dim=64, cache_type=mer_b200.VALUE_F16, page_tokens=16)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.install_attention(**{**good, **change})
    assert e.value.kind == INVALID
    c = Cache([(1, 4)], 8, 2, 64)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:  # and nothing is installed
        c.forward(backend, layer=5)
    assert e.value.kind == INVALID


def test_refused_lengths_of_host_arrays(backend):
    for kw in (dict(q_norm=np.ones(63)), dict(k_norm=np.ones((1, 64))), dict(sinks=np.ones(2))):
        with pytest.raises(ValueError):
            backend.install_attention(5, 8, 2, 64, mer_b200.VALUE_F16, 16, **kw)


@pytest.mark.parametrize("change", [dict(k_pages=None), dict(v_pages=None), dict(page_table=None), dict(row_start=None), dict(kv_len=None), dict(n_pages=0),
                                    dict(table_stride=0), dict(page_stride=4), dict(token_stride=68), dict(head_stride=8), dict(token_stride=0),
                                    dict(page_stride=1 << 62), dict(n_rows=1 << 31), "k", "table"])
def test_refused_batches(backend, change):
    c = Cache([(1, 4)], 8, 2, 64).fill().install(backend)
    x = torch.randn((1, 12 * 64), device="cuda", dtype=c.kind)
    rows = mer_b200.QkvRows(q=x.data_ptr(), k=x.data_ptr() + 1024, v=x.data_ptr() + 1280, q_out=c.out.data_ptr(), value_type=c.value_type)
    if change == "k":
        change = dict(k_pages=c.k.data_ptr() + 8)
    elif change == "table":
        change = dict(page_table=c.table.data_ptr() + 2)
    for call in (lambda b: backend.kv_append_device(0, b, rows), lambda b: backend.attention_forward_device(0, b, c.q.data_ptr(), c.out.data_ptr())):
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            call(c.batch(**change))
        assert e.value.kind == DISPATCH
    torch.cuda.synchronize()
    assert (c.out == 7.0).all()


def test_refused_rows(backend):
    c = Cache([(2, 4)], 8, 2, 64).fill().install(backend)
    x = torch.randn((2, 12 * 64), device="cuda", dtype=c.kind)
    good = dict(q=x.data_ptr(), k=x.data_ptr() + 1024, v=x.data_ptr() + 1280, q_out=c.out.data_ptr(), value_type=c.value_type)
    for change, kind in ((dict(k=None), INVALID), (dict(v=None), INVALID), (dict(q_out=None), INVALID), (dict(value_type=7), INVALID), (dict(q_stride=511), DISPATCH),
                         (dict(k_stride=127), DISPATCH), (dict(v_stride=1), DISPATCH), (dict(q_out_stride=500), DISPATCH), (dict(k=x.data_ptr() + 1), DISPATCH),
                         (dict(q_out=x.data_ptr(), q_stride=768), DISPATCH), (dict(q_out=x.data_ptr(), value_type=mer_b200.VALUE_F32), DISPATCH)):
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            backend.kv_append_device(0, c.batch(), mer_b200.QkvRows(**{**good, **change}))
        assert e.value.kind == kind, change
    for q, out, more, kind in ((None, c.out.data_ptr(), {}, INVALID), (c.q.data_ptr(), None, {}, INVALID), (c.q.data_ptr() + 2, c.out.data_ptr(), {}, DISPATCH),
                               (c.q.data_ptr(), c.out.data_ptr() + 8, {}, DISPATCH), (c.q.data_ptr(), c.out.data_ptr(), dict(q_stride=510), DISPATCH),
                               (c.q.data_ptr(), c.out.data_ptr(), dict(out_stride=516), DISPATCH)):
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            backend.attention_forward_device(0, c.batch(), q, out, 0, **more)
        assert e.value.kind == kind
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.attention_forward_device(77, c.batch(), c.q.data_ptr(), c.out.data_ptr())
    assert e.value.kind == INVALID
