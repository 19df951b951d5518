"""Keys and values quantised to 4 bits as they are written (mer_kv_append_device of a layer whose cache holds 4 bits), and rows read back
(mer_kv_read_device), against the definition in 64 bits.

Codes, scales and minima are equal: the kernel computes them in 64 bits, and what it can still have other than the reference is a value within
about 2^-48 of a border.  Values read back are one fma and one rounding of them: equal, too.  Queries: as with a cache of 16 bits (2^-19 of a
head's largest value, and one rounding)."""
import math

import numpy as np
import pytest

import mer_b200

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, mer_b200.VALUE_F32), "f16": (torch.float16, mer_b200.VALUE_F16), "bf16": (torch.bfloat16, mer_b200.VALUE_BF16)}
INVALID, DISPATCH = mer_b200.GpuExpertDispatchErrorKind.InvalidArgument, mer_b200.GpuExpertDispatchErrorKind.ValidationDispatch


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.fixture(scope="module")
def backend():
    with mer_b200.Backend(mer_b200.DTYPE_Q8_0, 64, 64, 1 << 20, 1, max_tokens=1, max_top_k=1) as b:
        yield b


def quantised(x, group):
    """Codes [..., d], scales and minima [..., groups] of 64-bit heads [..., d]."""
    codes, scales, minima = torch.zeros_like(x), [], []
    for a in range(0, x.shape[-1], group):
        part = x[..., a:a + group]
        lo, hi = part.amin(-1), part.amax(-1)
        odd = ~(part.abs() <= 60000.0).all(-1)
        least = lo.float().half()
        scale = ((hi - lo).float() * np.float32(1.0 / 15.0).item()).half()
        unit = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(scale, dtype=torch.float32)).double()
        code = ((part - least.double()[..., None]) * unit[..., None]).round().clamp(0, 15)
        least[odd], scale[odd] = math.nan, 0.0
        codes[..., a:a + group] = torch.where(odd[..., None], torch.zeros_like(code), code)
        scales.append(scale)
        minima.append(least)
    return codes, torch.stack(scales, -1), torch.stack(minima, -1)


def numbers(codes, scales, minima, group):
    """What they stand for, in 64 bits."""
    g = torch.arange(codes.shape[-1], device=codes.device) // group
    return codes * scales.double()[..., g] + minima.double()[..., g]


class Cache4:
    """Sequences of (new rows, tokens with them) in a pool of pages of 4 bits; what no sequence holds is bytes of any kind."""

    def __init__(self, lens, q_heads, kv_heads, d, kind="bf16", page=16, group=32, heads_first=False, seed=0, behind=0, wide=0, q_gap=0, gap=0):
        g = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.hq, self.hk, self.d, self.page, self.group = lens, q_heads, kv_heads, d, page, group
        self.kind, self.value_type = TYPES[kind]
        held = [-(-k // page) for _, k in lens]
        self.n_pages, widest = sum(held) + 2, max(held + [1]) + wide
        self.units = next(u for u in (2, 3, 4, 6, 8) if 32 * u >= d)
        self.groups = -(-32 * self.units // group)
        self.block = mer_b200.kv4_block_bytes(d, page, group)
        shape = (kv_heads, self.n_pages, self.block + gap) if heads_first else (self.n_pages, kv_heads, self.block + gap)
        self.pools = [torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g) for _ in range(2)]
        self.k, self.v = (p.transpose(0, 1) if heads_first else p for p in self.pools)
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
        self.opts = {}

    def places(self, i, first=0, last=None):
        at = torch.arange(first, self.lens[i][1] if last is None else last, device="cuda")
        return self.table[i, at // self.page].long(), at % self.page

    def parts(self, keys):
        """Views: words of codes [page, head, token, words], scales and minima [page, head, token, groups, 2]."""
        pages, size = (self.k if keys else self.v), self.page * 16 * self.units
        return (pages[..., :size].view(torch.int32 if keys else torch.int16).unflatten(-1, (self.page, -1)),
                pages[..., size:size + self.page * 4 * self.groups].view(torch.float16).unflatten(-1, (self.page, self.groups, 2)))

    def order(self, keys):
        """For each word and nibble of a token the value it holds."""
        v = torch.arange(32 * self.units, device="cuda")
        word, bit = ((v % 32 // 8) * self.units + v // 32, v % 8 // 2 * 4 + v % 2 * 16) if keys else ((v % 32 // 4) * self.units + v // 32, v % 4 * 4)
        return word, bit

    def put(self, keys, places, codes, scales, minima):
        """Codes [tokens, heads, d] and so on into pages and slots; zeros behind the head's own values."""
        words, numbers_ = self.parts(keys)
        word, bit = self.order(keys)
        full = torch.zeros((*codes.shape[:-1], 32 * self.units), dtype=torch.int64, device="cuda")
        full[..., :self.d] = codes.to(torch.int64)
        made = torch.zeros((*codes.shape[:-1], words.shape[-1]), dtype=torch.int64, device="cuda")
        made.index_add_(-1, word, full << bit)
        words[places[0], :, places[1]] = made.to(words.dtype)
        pair = torch.zeros((*scales.shape[:-1], self.groups, 2), dtype=torch.float16, device="cuda")
        pair[..., :scales.shape[-1], 0], pair[..., :scales.shape[-1], 1] = scales, minima
        numbers_[places[0], :, places[1]] = pair

    def held(self, keys, places):
        """What the cache has there, in 64 bits: [tokens, heads, d]."""
        words, numbers_ = self.parts(keys)
        word, bit = self.order(keys)
        codes = (words[places[0], :, places[1]].to(torch.int64)[..., word] >> bit & 15)[..., :self.d]
        pair = numbers_[places[0], :, places[1]].double()
        g = torch.arange(self.d, device="cuda") // self.group
        return codes.double() * pair[..., g, 0] + pair[..., g, 1]

    def fill(self, first=None, scale=1.0):
        """Tokens of every sequence (from first[i] on)."""
        for i, (_, k) in enumerate(self.lens):
            lo = 0 if first is None else first[i]
            if k > lo:
                for keys in (True, False):
                    x = torch.randn((k - lo, self.hk, self.d), device="cuda", generator=self.gen).double() * scale
                    self.put(keys, self.places(i, lo), *quantised(x, self.group))
        return self

    def batch(self, **kw):
        f = dict(k_pages=self.k.data_ptr(), v_pages=self.v.data_ptr(), n_pages=self.n_pages, page_stride=self.k.stride(0), head_stride=self.k.stride(1),
                 page_table=self.table.data_ptr(), table_stride=self.table.shape[1], row_start=self.row_start.data_ptr(),
                 kv_len=self.kv_len.data_ptr(), n_seqs=len(self.lens), n_rows=self.rows)
        return mer_b200.KvBatch(**{**f, **kw})

    def install(self, b, layer=0, **kw):
        b.install_attention(layer, self.hq, self.hk, self.d, self.value_type, self.page, cache_bits=4, cache_group=self.group, **kw)
        self.opts = kw
        return self


LENS = {
    "one": [(1, 1)],
    "decode": [(1, 77), (1, 1), (1, 300), (1, 16), (1, 129)],
    "idle": [(0, 40), (1, 33), (0, 0), (0, 5), (1, 90), (0, 7)],
    "prompts": [(33, 33), (100, 257), (1, 50), (200, 200)],
}


def exact_rows(c, x, qw, kw, freq, pairs, eps, rope_scale=1.0):
    """Norm and rotation of rows [rows, heads, d] in 64 bits."""
    exact, r = x.double().clone(), 2 * len(freq)
    for a, b, w in ((0, c.hq, qw), (c.hq, c.hq + c.hk, kw)):
        if w is not None:
            part = exact[:, a:b]
            exact[:, a:b] = part / (part.square().mean(2, keepdim=True) + eps).sqrt() * torch.tensor(w, dtype=torch.float64, device="cuda")
    if r:
        pos = torch.cat([torch.arange(k - n, k, dtype=torch.float64) for n, k in c.lens]).cuda()
        angle = (pos[:, None] * torch.tensor(freq, device="cuda"))[:, None]
        cos, sin = angle.cos() * rope_scale, angle.sin() * rope_scale
        i, j = (slice(0, r, 2), slice(1, r, 2)) if pairs else (slice(0, r // 2), slice(r // 2, r))
        a, b = exact[:, :c.hq + c.hk, i].clone(), exact[:, :c.hq + c.hk, j].clone()
        exact[:, :c.hq + c.hk, i], exact[:, :c.hq + c.hk, j] = a * cos - b * sin, a * sin + b * cos
    return exact


def append(b, c, source="bf16", *, norm=True, rope_dims=0, pairs=False, theta=1e4, rope_scale=1.0, gap=0, offset=0, with_q=True, x=None, eps=1e-5):
    """Appends rows; the rows in 64 bits as they come out of norm and rotation."""
    dtype, value_type = TYPES[source]
    width = (c.hq + 2 * c.hk) * c.d
    store = torch.randn(c.rows * (width + gap) + offset, device="cuda", generator=c.gen).mul_(2).to(dtype)
    rows = store[offset:].view(c.rows, width + gap)
    if x is not None:
        rows[:, :width] = x
    rng = np.random.default_rng(9)
    qw, kw = ((1 + 0.3 * rng.standard_normal(c.d)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    freq = theta ** (-np.arange(rope_dims // 2) / max(1, rope_dims // 2))
    eps = float(np.float32(eps))
    c.install(b, q_norm=qw, k_norm=kw, norm_eps=eps, rope_freq=freq if rope_dims else None, rope_pairs=pairs, rope_scale=rope_scale)
    at = rows.data_ptr()
    size = dtype.itemsize
    b.kv_append_device(0, c.batch(), mer_b200.QkvRows(q=at if with_q else None, k=at + c.hq * c.d * size, v=at + (c.hq + c.hk) * c.d * size,
                                                      q_out=c.out.data_ptr() if with_q else None, q_stride=width + gap, k_stride=width + gap,
                                                      v_stride=width + gap, value_type=value_type), stream())
    return exact_rows(c, rows[:c.starts[-1], :width].reshape(-1, c.hq + 2 * c.hk, c.d), qw, kw, freq, pairs, eps, float(np.float32(rope_scale)))


def check_append(b, c, source="bf16", **kw):
    before = [p.clone() for p in c.pools]
    exact = append(b, c, source, **kw)
    b.stream_check(0, stream())
    after = [p.clone() for p in c.pools]
    for p, q in zip(c.pools, before):
        p.copy_(q)
    for keys, a in ((True, c.hq), (False, c.hq + c.hk)):
        for i, (n, k) in enumerate(c.lens):
            if n:
                c.put(keys, c.places(i, k - n), *quantised(exact[c.starts[i]:c.starts[i + 1], a:a + c.hk], c.group))
    for p, q, name in zip(c.pools, after, "kv"):  # every byte: codes, scales, minima, and what belongs to nobody
        assert torch.equal(p, q), (name, (p != q).nonzero()[:5])
    if kw.get("with_q", True):
        q, want = c.out[:c.starts[-1]].double().view(-1, c.hq, c.d), exact[:, :c.hq]
        bound = (torch.finfo(c.kind).eps / 2 + 2.0 ** -19) * want.abs() + 2.0 ** -19 * want.abs().amax(2, keepdim=True) + 2.0 ** -25
        assert ((q - want).abs() <= bound).all()
    assert (c.out[c.starts[-1]:] == 7.0).all()
    return exact


@pytest.mark.parametrize("source", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,d,kind,page,group,rope_dims,pairs,norm", [
    (32, 4, 128, "bf16", 16, 32, 128, False, True), (8, 8, 128, "f16", 24, 64, 64, True, False), (6, 6, 64, "bf16", 1, 32, 64, False, True), (20, 4, 80, "f16", 24, 64, 40, True, True),
    (20, 4, 80, "bf16", 5, 32, 20, False, True), (2, 1, 8, "bf16", 3, 32, 8, False, True), (3, 3, 96, "f16", 40, 32, 96, False, True), (4, 2, 256, "bf16", 16, 64, 256, False, True),
    (7, 1, 136, "f16", 5, 32, 10, False, True), (3, 1, 24, "bf16", 16, 64, 0, False, True), (5, 5, 200, "bf16", 128, 64, 200, True, True), (4, 1, 192, "f16", 8, 32, 192, False, False),
    (1, 1, 160, "bf16", 16, 64, 144, False, True), (12, 3, 64, "f16", 16, 64, 48, False, True)])
def test_append(backend, source, q_heads, kv_heads, d, kind, page, group, rope_dims, pairs, norm):
    for lens in LENS.values():
        c = Cache4(lens, q_heads, kv_heads, d, kind, page, group, behind=3, gap=32)
        check_append(backend, c, source, norm=norm, rope_dims=rope_dims, pairs=pairs)


@pytest.mark.parametrize("offset,gap", [(1, 0), (4, 12), (0, 3), (8, 8)])
def test_append_rows_at_odd_places(backend, offset, gap):
    for source in TYPES:
        c = Cache4(LENS["prompts"], 4, 2, 64, "bf16", 16, heads_first=True)
        check_append(backend, c, source, rope_dims=32, offset=offset, gap=gap)


def test_append_many_rows_far_positions_and_sequences(backend):
    check_append(backend, Cache4([(3000, 3000), (1, 70), (2500, 9000)], 2, 2, 128, "f16", 64, seed=4), "f16", rope_dims=128, theta=1e6, rope_scale=1.3)
    rng = np.random.default_rng(5)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 3, 3000), rng.integers(0, 40, 3000))]
    check_append(backend, Cache4(lens, 2, 1, 64, "bf16", 8, seed=2, behind=5), "bf16", rope_dims=64)
    c = Cache4([(2, 5_000_000)], 2, 2, 64, "bf16", 1 << 20)  # angles of millions
    check_append(backend, c, "f32", rope_dims=64, with_q=False)


def test_groups_of_every_kind(backend):
    # equal values, zeros, one value apart, tiny and large ones, ties between two codes
    c = Cache4([(8, 20)], 1, 1, 128, "bf16", 16)
    x = torch.randn((8, 3 * 128), device="cuda", generator=c.gen)
    x[0] = 0.0
    x[1] = 3.25
    x[2] = 1e-7 * torch.randn(384, device="cuda", generator=c.gen)
    x[3] = 30000.0 * torch.randn(384, device="cuda", generator=c.gen).clamp(-1.9, 1.9)
    x[4] = torch.arange(384, device="cuda") % 32 / 2.0  # halves of a step of 31 / 30
    x[5] = torch.tensor([0.0, 15.0] + [i / 2 for i in range(30)], device="cuda").repeat(12)  # scale 1: ties go to the even code
    x[6] = 1000.0 + 0.01 * torch.randn(384, device="cuda", generator=c.gen)
    x[7, ::32] = 60000.0
    for group in (32, 64):
        c = Cache4([(8, 20)], 1, 1, 128, "bf16", 16, group)
        check_append(backend, c, "f32", norm=False, x=x)


@pytest.mark.parametrize("size,eps", [(1e18, 1e-5), (1e25, 1e-5), (1e37, 0.0), (1e-14, 0.0), (1e-17, 0.0), (1e-21, 0.0), (1e-30, 0.0), (1e-21, 1e-40)])
def test_norms_of_rows_far_from_one(backend, size, eps):
    # the sum of squares leaves 32 bits' range; the codes are those of 64 all the same
    c = Cache4([(5, 9), (1, 30)], 2, 2, 128, "bf16", 16)
    x = torch.randn((6, 6 * 128), device="cuda", generator=c.gen)
    x[:, 256:512] *= size
    exact = check_append(backend, c, "f32", rope_dims=64, with_q=False, x=x, eps=eps)
    assert exact[:, 2:4].isfinite().all() and exact[:, 2:4].abs().max() > 0.1  # the oracle's own: 1e-21 a value over the root of 1e-40 + 1e-42 is 0.1


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("q_heads,kv_heads,d,lens,gap,offset", [(32, 4, 128, [(1, 100)], 0, 0), (20, 2, 80, [(3, 3), (0, 9), (1, 17)], 8, 0), (5, 5, 64, [(40, 77)], 3, 1), (64, 8, 256, [(2, 2)], 0, 0),
                                                              (4, 2, 24, [(3000, 3000)], 0, 8)])
def test_queries_in_place(backend, q_heads, kv_heads, d, lens, gap, offset, pairs):
    # one warp a row, and several of them that each have some of its heads
    got = {}
    for place in ("own", "same"):
        c = Cache4(lens, q_heads, kv_heads, d, "bf16", 16)
        width, rope = (q_heads + 2 * kv_heads) * d + gap, d // 4 * 2
        rows = torch.randn(c.rows * width + offset, device="cuda", generator=c.gen).to(torch.bfloat16)[offset:].view(c.rows, width)
        kept = rows.clone()
        q_out = rows if place == "same" else torch.zeros_like(rows)
        norm = (1 + 0.3 * np.random.default_rng(3).standard_normal(d)).astype(np.float32)
        c.install(backend, q_norm=norm, k_norm=norm, norm_eps=1e-5, rope_freq=1e4 ** (-np.arange(rope // 2) / (rope // 2)), rope_pairs=pairs)
        at = rows.data_ptr()
        backend.kv_append_device(0, c.batch(), mer_b200.QkvRows(q=at, k=at + q_heads * d * 2, v=at + (q_heads + kv_heads) * d * 2, q_out=q_out.data_ptr(), q_stride=width, k_stride=width,
                                                                v_stride=width, q_out_stride=width, value_type=mer_b200.VALUE_BF16), stream())
        backend.stream_check(0, stream())
        assert torch.equal(rows[:, q_heads * d:], kept[:, q_heads * d:]) and (place == "same" or torch.equal(rows, kept))
        got[place] = [q_out[:, :q_heads * d].clone(), *(p.clone() for p in c.pools)]
    assert all(torch.equal(a, b) for a, b in zip(got["own"], got["same"]))


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, 60001.0, -1e30])
def test_values_that_a_group_has_no_room_for(backend, what):
    c = Cache4([(4, 20), (3, 3)], 2, 2, 128, "bf16", 16)
    x = torch.randn((7, 6 * 128), device="cuda", generator=c.gen)
    x[2, 2 * 128 + 40] = what   # row 2, key head 0, group 1
    x[5, 5 * 128 + 127] = what  # row 5, value head 1, group 3
    exact = check_append(backend, c, "f32", norm=False, x=x)
    k, v = read(backend, c, "f32")
    assert torch.isnan(k.view(7, 2, 128)[2, 0, 32:64]).all() and torch.isnan(v.view(7, 2, 128)[5, 1, 96:]).all()
    k.view(7, 2, 128)[2, 0, 32:64] = 0
    v.view(7, 2, 128)[5, 1, 96:] = 0
    assert torch.isfinite(k).all() and torch.isfinite(v).all() and exact.isfinite().sum() >= 7 * 6 * 128 - 2


def read(b, c, kind="f32", k=True, v=True, gap=0, offset=0, layer=0, **kw):
    dtype, value_type = TYPES[kind]
    width = c.hk * c.d
    stores = [torch.full((c.rows * (width + gap) + offset,), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    rows = [s[offset:].view(c.rows, width + gap) for s in stores]
    b.kv_read_device(layer, c.batch(**kw), mer_b200.KvRows(k=rows[0].data_ptr() if k else None, v=rows[1].data_ptr() if v else None, k_stride=width + gap, v_stride=width + gap,
                                                           value_type=value_type), stream())
    return rows


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv_heads,d,page,group,gap,offset", [(4, 128, 16, 32, 0, 0), (1, 64, 1, 64, 0, 0), (8, 80, 24, 32, 0, 0), (3, 8, 3, 32, 5, 1), (2, 256, 64, 64, 8, 0), (5, 136, 5, 64, 0, 4),
                                                            (40, 96, 16, 32, 0, 0), (2, 192, 256, 32, 0, 0)])
def test_rows_read_back(backend, kind, kv_heads, d, page, group, gap, offset):
    dtype = TYPES[kind][0]
    for lens in (*LENS.values(), [(700, 700), (0, 9), (1, 1), (2000, 2100)]):
        c = Cache4(lens, kv_heads, kv_heads, d, "bf16", page, group, behind=2, heads_first=d == 80).fill().install(backend)
        rows = read(backend, c, kind, gap=gap, offset=offset)
        backend.stream_check(0, stream())
        for got, keys in zip(rows, (True, False)):
            for i, (n, k) in enumerate(lens):
                want = c.held(keys, c.places(i, k - n)).float().to(dtype) if n else None
                if n:
                    assert torch.equal(got[c.starts[i]:c.starts[i + 1], :kv_heads * d].reshape(n, kv_heads, d), want), (i, keys)
            assert (got[c.starts[-1]:] == 7.0).all() and (got[:, kv_heads * d:] == 7.0).all()


def test_read_one_of_the_two(backend):
    c = Cache4(LENS["prompts"], 2, 2, 64).fill().install(backend)
    both = read(backend, c)
    for k in (True, False):
        one = read(backend, c, k=k, v=not k)
        assert torch.equal(one[0 if k else 1], both[0 if k else 1]) and (one[1 if k else 0] == 7.0).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_rows_of_a_cache_of_16_bits(backend, kind, cache):
    from test_gpu_attention import Cache
    for heads_first, d, page in ((False, 64, 16), (True, 80, 5), (False, 256, 24)):
        c = Cache(LENS["prompts"], 4, 2, d, cache, page, heads_first=heads_first, behind=2).fill().install(backend, layer=3)
        rows = read(backend, c, kind, layer=3)
        for got, pages in zip(rows, (c.k, c.v)):
            for i, (n, k) in enumerate(c.lens):
                assert torch.equal(got[c.starts[i]:c.starts[i + 1]].reshape(n, 2, d), pages[c.places(i, k - n)].float().to(TYPES[kind][0]))
            assert (got[c.starts[-1]:] == 7.0).all()


def test_append_then_read_is_the_nearest_code(backend):
    c = Cache4([(500, 500), (1, 80)], 2, 2, 128, "bf16", 16)
    exact = append(backend, c, "f32", rope_dims=128)
    k, v = read(backend, c)
    for got, a in ((k, 2), (v, 4)):
        x = exact[:, a:a + 2]
        step = quantised(x, 32)[1].double().repeat_interleave(32, -1)
        # half a step, the codes' ends a scale's and a minimum's rounding (2^-11 of 15 steps and of the smallest value) further out
        bound = step * (0.5 + 15 * 2.0 ** -11) + x.abs().amax(-1, keepdim=True) * 2.0 ** -11 + 2.0 ** -23
        assert ((got.view(-1, 2, 128).double() - x).abs() <= bound).all()


# ------------------------------------------------------------------------------------------------ calls that go wrong


def test_rows_without_a_place(backend):
    c = Cache4([(2, 50), (6, 4), (3, 0), (1, 20)], 2, 2, 64).fill().install(backend)
    good = read(backend, c)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.stream_check(0, stream())
    assert e.value.kind == DISPATCH
    backend.stream_check(0, stream())  # reported once
    for x, keys in zip(good, (True, False)):
        assert (x[2:4] == 0).all() and (x[8:11] == 0).all()
        assert torch.equal(x[4:8].view(4, 2, 64), c.held(keys, c.places(1)).float())
        assert torch.equal(x[11:].view(1, 2, 64), c.held(keys, c.places(3, 19)).float())
    before = [p.clone() for p in c.pools]
    store = torch.randn((12, 6 * 64), device="cuda", generator=c.gen).to(c.kind)
    at = store.data_ptr()
    backend.kv_append_device(0, c.batch(), mer_b200.QkvRows(k=at, v=at + 256, k_stride=384, v_stride=384, value_type=c.value_type), stream())
    with pytest.raises(mer_b200.GpuExpertDispatchError):
        backend.stream_check(0, stream())
    after = [p.clone() for p in c.pools]
    for p, q in zip(c.pools, before):
        p.copy_(q)
    for keys, x in ((True, store[:, :128]), (False, store[:, 128:256])):
        for i, rows, first in ((0, slice(0, 2), 48), (1, slice(4, 8), 0), (3, slice(11, 12), 19)):
            c.put(keys, c.places(i, first), *quantised(x[rows].double().view(-1, 2, 64), 32))
    assert all(torch.equal(p, q) for p, q in zip(c.pools, after))


@pytest.mark.parametrize("wrong", ["number", "table"])
def test_pages_that_are_not_there(backend, wrong):
    c = Cache4([(100, 100), (180, 200), (60, 60)], 2, 2, 64).fill().install(backend)
    good = read(backend, c)
    if wrong == "number":
        c.table[1, 3], c.table[1, 5] = c.n_pages, -1
        bad = torch.cat([torch.arange(48, 64), torch.arange(80, 96)]) + 80  # tokens 48 .. and 80 .. of the rows from token 20 on
        rows = read(backend, c)
    else:
        narrow = c.table[:, :7].contiguous()  # 112 tokens: sequence 1 has more
        bad = torch.arange(100, 280)
        rows = read(backend, c, page_table=narrow.data_ptr(), table_stride=7)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.stream_check(0, stream())
    assert e.value.kind == DISPATCH
    for x, y in zip(rows, good):
        assert (x[bad] == 0).all()
        x[bad] = y[bad]
        assert torch.equal(x, y)


def test_offsets_beyond_32_bits(backend):
    # two pages five gigabytes apart
    page, d, hk = 16, 128, 2
    block = mer_b200.kv4_block_bytes(d, page)
    pool = torch.zeros(5 * (1 << 30) + 4 * block, dtype=torch.uint8, device="cuda")
    c = Cache4([(20, 32)], 2, hk, d, "bf16", page)
    far = 5 * (1 << 30) // 16 * 16
    c.n_pages, c.table = 2, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    views = [torch.as_strided(pool, (2, hk, block), (far, block, 1), i * 2 * block) for i in range(2)]
    c.k, c.v, c.pools = views[0], views[1], views
    check_append(backend, c, "bf16", rope_dims=128, with_q=False)
    rows = read(backend, c)
    for got, keys in zip(rows, (True, False)):
        assert torch.equal(got.view(20, hk, d), c.held(keys, c.places(0, 12)).float())


def test_empty_batches(backend):
    c = Cache4([(1, 4)], 2, 2, 64).fill().install(backend)
    before = [p.clone() for p in c.pools]
    for kw in (dict(n_rows=0), dict(n_seqs=0)):
        rows = read(backend, c, **kw)
        assert all((x == 7.0).all() for x in rows)
    assert all(torch.equal(p, q) for p, q in zip(c.pools, before))


def test_captured_calls_follow_their_tables(backend):
    c = Cache4([(1, 40), (3, 60), (2, 2)], 4, 2, 128, "bf16", 16, behind=4)
    x = torch.randn((c.rows, 8 * 128), device="cuda", generator=c.gen).to(c.kind)
    c.install(backend, rope_freq=np.ones(64) * 0.01)
    at = x.data_ptr()
    qkv = mer_b200.QkvRows(q=at, k=at + 1024, v=at + 1536, q_out=c.out.data_ptr(), q_stride=1024, k_stride=1024, v_stride=1024, value_type=c.value_type)
    out = [torch.zeros((c.rows, 256), dtype=torch.float32, device="cuda") for _ in range(2)]
    kv = mer_b200.KvRows(k=out[0].data_ptr(), v=out[1].data_ptr(), value_type=mer_b200.VALUE_F32)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        backend.kv_append_device(0, c.batch(), qkv, side.cuda_stream)
        backend.kv_read_device(0, c.batch(), kv, side.cuda_stream)
    for lens in ([(1, 40), (3, 60), (2, 2)], [(5, 33), (0, 60), (1, 16)]):
        c.lens, starts = lens, np.cumsum([0] + [n for n, _ in lens]).tolist()
        c.starts = starts
        c.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
        c.kv_len.copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        exact = exact_rows(c, x[:starts[-1]].view(-1, 8, 128), None, None, np.ones(64) * 0.01, False, 0.0)
        for got, a in zip(out, (4, 6)):
            assert torch.equal(got[:starts[-1]].view(-1, 2, 128).double(), numbers(*quantised(exact[:, a:a + 2], 32), 32).float().double())


@pytest.mark.parametrize("change", [dict(cache_group=16), dict(cache_group=128), dict(cache_group=33), dict(head_dim=12), dict(cache_type=mer_b200.VALUE_F32)])
def test_refused_layers(backend, change):
    good = dict(layer=9, q_heads=8, kv_heads=2, head_dim=64, cache_type=mer_b200.VALUE_F16, page_tokens=16, cache_bits=4)
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.install_attention(**{**good, **change})
    assert e.value.kind == INVALID
    with pytest.raises(ValueError):
        backend.install_attention(**{**good, "cache_bits": 8})


@pytest.mark.parametrize("change", [dict(k_pages=None), dict(v_pages=None), dict(page_table=None), dict(row_start=None), dict(kv_len=None), dict(n_pages=0), dict(table_stride=0),
                                    dict(page_stride=8), dict(token_stride=80), dict(head_stride=24), dict(head_stride=16), dict(page_stride=1 << 62), dict(n_rows=1 << 31), "k", "table"])
def test_refused_batches(backend, change):
    c = Cache4([(1, 4)], 8, 2, 64).fill().install(backend)
    x = torch.randn((1, 12 * 64), device="cuda").to(c.kind)
    rows = mer_b200.QkvRows(q=x.data_ptr(), k=x.data_ptr() + 1024, v=x.data_ptr() + 1280, q_out=c.out.data_ptr(), value_type=c.value_type)
    out = torch.full((1, 128), 7.0, device="cuda")
    change = dict(k_pages=c.k.data_ptr() + 8) if change == "k" else dict(page_table=c.table.data_ptr() + 2) if change == "table" else change
    before = [p.clone() for p in c.pools]
    for call in (lambda b: backend.kv_append_device(0, b, rows), lambda b: backend.attention_forward_device(0, b, c.q.data_ptr(), c.out.data_ptr()),
                 lambda b: backend.kv_read_device(0, b, mer_b200.KvRows(k=out.data_ptr(), value_type=mer_b200.VALUE_F32))):
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            call(c.batch(**change))
        assert e.value.kind == DISPATCH
    torch.cuda.synchronize()
    assert (c.out == 7.0).all() and (out == 7.0).all() and all(torch.equal(p, q) for p, q in zip(c.pools, before))


def test_refused_rows_to_read(backend):
    c = Cache4([(2, 4)], 8, 2, 64).fill().install(backend)
    out = torch.full((4, 136), 7.0, device="cuda")
    for change, kind in ((dict(k=None, v=None), INVALID), (dict(value_type=3), INVALID), (dict(k_stride=127), DISPATCH), (dict(v_stride=100), DISPATCH), (dict(k=out.data_ptr() + 2), DISPATCH),
                         (dict(k_stride=1 << 41), DISPATCH)):
        with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
            backend.kv_read_device(0, c.batch(), mer_b200.KvRows(**{**dict(k=out.data_ptr(), v=out.data_ptr(), value_type=mer_b200.VALUE_F32), **change}))
        assert e.value.kind == kind, change
    with pytest.raises(mer_b200.GpuExpertDispatchError) as e:
        backend.kv_read_device(77, c.batch(), mer_b200.KvRows(k=out.data_ptr(), value_type=mer_b200.VALUE_F32))
    assert e.value.kind == INVALID
    torch.cuda.synchronize()
    assert (out == 7.0).all()
