"""Performance cases of the attention side of a decoder layer, measured through the package's public entry points.

  append   the rows of a layer's fused q|k|v projection: RMSNorm of every query and key head, the position rotation, keys and
           values into the pages of a paged cache, queries out in the cache's type (kv_append_device)
  attend   the new rows' queries over the keys and values of their sequences in the paged cache (attention_forward_device)

A batch holds sequences of different lengths.  Sequence s brings rows row_start[s] .. row_start[s + 1] of the batch, its
newest tokens, and has kv_len[s] tokens in the cache with them; its page table says where.  `pattern` says how many rows:

  decode   one each
  draft    `rows` each: a draft model's tokens to be verified
  prompts  between rows / 2 and rows each
  mixed    the first sequence `rows`, a chunk of its prompt, the others one each

and a sequence has between ctx_lo and ctx_hi tokens from before (by their logarithm).  `idle` sequences more bring no row."""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MAX_SCORES = 2.2e9  # of a drawn case's plain form: the largest listed one has 2.1e9
MAX_KEYS = 3.2e8    # values of the keys that a drawn case's plain form lays out: the largest listed one has 2.7e8
MAX_FLOPS, MAX_BYTES = 1.0e12, 6.0e8  # of a drawn case: the longest listed one does 1.06e12 (and takes ten times as long as moving the bytes)
EPS = 1e-6

_BASE = dict(kind="attend", q_heads=32, kv_heads=4, head_dim=128, cache="bf16", page=16, heads_first=False, pattern="decode", seqs=1,
             rows=1, idle=0, ctx_lo=0, ctx_hi=0, lens=0)
_APPEND = dict(source="bf16", norm=True, pairs=False, rope_dims=128, theta=1e6)
_ATTEND = dict(window=0, sinks=False, sharp=1.0)


def _case(**kw):
    c = {**_BASE, **(_APPEND if kw.get("kind") == "append" else _ATTEND)}
    unknown = set(kw) - set(c) - {"name"}
    assert not unknown, unknown
    return {**c, **kw}


_MANY = dict(q_heads=32, kv_heads=4, head_dim=128)  # heads of the 128-expert layers
_FEW = dict(q_heads=32, kv_heads=8, head_dim=128)   # heads of the 8-expert layers


def listed():
    return [
        # One user's token: the smallest call there is, launch and latency.
        _case(name="append-decode-b1", kind="append", ctx_lo=900, ctx_hi=900, **_MANY),
        # A serving batch whose projection left 32-bit rows, as the expert layers take and give them; far positions.
        _case(name="append-decode-b64-f32", kind="append", source="f32", seqs=64, ctx_lo=500, ctx_hi=16000, lens=1, **_MANY),
        # A prompt of 2048 tokens on its way into the cache.
        _case(name="append-prompt-2048", kind="append", pattern="prompts", rows=2048, **_MANY),
        # Many prompts of odd lengths at once: no norms, neighbouring values rotated, half of a head, pages that are no power of two.
        _case(name="append-ragged-f16", kind="append", cache="f16", source="f16", norm=False, pairs=True, rope_dims=64, theta=1e4, page=24,
              heads_first=True, pattern="prompts", seqs=13, rows=1333, idle=1, ctx_lo=1, ctx_hi=700, lens=2, **_FEW),
        # One user's token far into a long text: few rows, a long axis to split.
        _case(name="attend-decode-b1-32k", ctx_lo=32000, ctx_hi=32000, **_MANY),
        # A serving batch of 64 users with contexts of very different lengths.
        _case(name="attend-decode-b64", seqs=64, ctx_lo=800, ctx_hi=8000, lens=3, page=32, **_MANY),
        # A window of 128 tokens, a learned sink for each head, heads of 64: little to read, so latency counts.
        _case(name="attend-decode-window-b16", q_heads=64, kv_heads=8, head_dim=64, seqs=16, ctx_lo=100, ctx_hi=4000, lens=4, window=128,
              sinks=True),
        # Drafts of five tokens for eight users.
        _case(name="attend-draft-b8", cache="f16", pattern="draft", seqs=8, rows=5, ctx_lo=1000, ctx_hi=6000, lens=5, sharp=2.0, **_FEW),
        # A prompt of 2048 tokens from its start.
        _case(name="attend-prompt-2048", pattern="prompts", rows=2048, page=64, **_MANY),
        # A chunk of a prompt and 47 users' single tokens in one step.
        _case(name="attend-mixed-b48", pattern="mixed", seqs=48, rows=777, idle=1, ctx_lo=300, ctx_hi=6000, lens=6, page=32, sharp=2.0, **_FEW),
        # A few prompts at once with an odd head size and an odd number of query heads for each key head.
        _case(name="attend-prompts-d80", cache="f16", q_heads=20, kv_heads=4, head_dim=80, pattern="prompts", seqs=4, rows=700, ctx_lo=50,
              ctx_hi=900, lens=7, page=24, heads_first=True),
        # The largest call: a chunk of 2048 tokens behind 30 thousand that are in the cache.
        _case(name="attend-chunk-2048-30k", pattern="prompts", rows=2048, ctx_lo=30700, ctx_hi=30700, page=64, **_MANY),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kv_heads = rng.choice([1, 2, 4, 4, 8, 8])
        c = dict(kind=rng.choice(["append", "attend", "attend"]), kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 8, 16]),
                 head_dim=rng.choice([64, 64, 128, 128, 128, 128, 80, 96, 256]), cache=rng.choice(["bf16", "bf16", "f16"]),
                 page=rng.choice([16, 16, 32, 64, 128, 256, 1, 24, 40]), heads_first=rng.random() < 0.3,
                 pattern=rng.choice(["decode", "decode", "draft", "prompts", "prompts", "mixed"]), idle=rng.choice([0, 0, 1, 2]), lens=rng.randrange(1 << 20))
        if c["pattern"] == "decode":
            c.update(seqs=_log_int(rng, 1, 200))
        elif c["pattern"] == "draft":
            c.update(seqs=_log_int(rng, 1, 48), rows=rng.randint(2, 9))
        elif c["pattern"] == "prompts":
            c.update(seqs=_log_int(rng, 1, 8), rows=_log_int(rng, 16, 4096))
        else:
            c.update(seqs=_log_int(rng, 2, 64), rows=_log_int(rng, 16, 2048))
        c["ctx_lo"] = _log_int(rng, 1, 8000) if c["pattern"] != "prompts" or rng.random() < 0.5 else 0
        c["ctx_hi"] = min(32000, c["ctx_lo"] * rng.randint(1, 10))
        if c["kind"] == "append":
            d = c["head_dim"]
            c.update(source=rng.choice(["bf16", "f32", "f16"]), norm=rng.random() < 0.6, pairs=rng.random() < 0.3, rope_dims=rng.choice([d, d, d, d // 2, 0]),
                     theta=rng.choice([1e4, 1e6, 5e5]))
        else:
            c.update(window=rng.choice([0, 0, 0, 128, 1024, rng.randint(1, 3000)]), sinks=rng.random() < 0.25, sharp=rng.choice([1.0, 2.0]))
        c = _case(**c)
        w, lens = work(c), lengths(c)
        scores = sum(n * k for n, k in _padded(lens)) * c["q_heads"]
        keys = sum(k for n, k in lens) * kv_heads * c["head_dim"]
        laid_out = max(s * k for s, _, k in _groups(lens)) * kv_heads * c["head_dim"]
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and keys <= MAX_KEYS and (c["kind"] == "append" or (scores <= MAX_SCORES and laid_out <= MAX_KEYS)):
            return c


def lengths(case):
    """(new rows, tokens in the cache with them) of each sequence: part of the case, whatever the seed."""
    c, rng = case, random.Random(case["lens"])
    got = []
    for s in range(c["seqs"] + c["idle"]):
        ctx = 0 if c["ctx_hi"] == 0 else _log_int(rng, max(1, c["ctx_lo"]), max(1, c["ctx_hi"]))
        n = {"decode": 1, "draft": c["rows"], "mixed": c["rows"] if s == 0 else 1}.get(c["pattern"])
        if n is None:
            n = c["rows"] if c["seqs"] == 1 else rng.randint(max(1, c["rows"] // 2), c["rows"])
        got.append((0 if s >= c["seqs"] else n, ctx + n))
    rng.shuffle(got)
    return got


def _groups(lens):
    """(sequences, rows, longest context) of the sequences that bring equally many rows: what the plain form computes at once."""
    by = {}
    for n, k in lens:
        if n:
            by.setdefault(n, []).append(k)
    return [(len(v), n, max(v)) for n, v in by.items()]


def _padded(lens):
    return [(s * n, k) for s, n, k in _groups(lens)]


def work(case):
    c, lens = case, lengths(case)
    rows, tables = sum(n for n, _ in lens), 4 * len(lens) * 2
    hq, hk, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "append":
        size = TYPES[c["source"]].itemsize
        return {"bytes": rows * (hq + 2 * hk) * d * (size + 2) + tables, "flops": rows * (hq + hk) * d * (4.0 * c["norm"] + 3.0)}
    pairs = seen = 0
    for n, k in lens:
        w = c["window"] or k
        full = max(0, min(n, w - (k - n) - 1))  # rows whose window reaches before the first token
        first = k - n + 1
        pairs += full * first + full * (full - 1) // 2 + (n - full) * w if c["window"] else n * first + n * (n - 1) // 2
        seen += min(k, w + n - 1) if n else 0
    return {"bytes": rows * hq * d * 4 + seen * hk * d * 4 + tables, "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------ inputs


class _State:
    pass


def _generator(seed, tag):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + tag + 1) % (1 << 62))


def _randn(shape, gen, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.view(-1).split(1 << 27):  # no second copy of a large cache in 32 bits
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen).mul_(scale))
    return out


def prepare(case, seed):
    c, s = case, _State()
    s.case, s.lens = c, lengths(c)
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    kind, gen = TYPES[c["cache"]], _generator(seed, 1)
    s.rows = sum(n for n, _ in s.lens)
    # the cache: a pool of pages, of which each sequence has some in any order
    held = [-(-k // page) for _, k in s.lens]
    n_pages, widest = sum(held) + 3, max(held)
    shape = (n_pages, hk, page, d) if c["heads_first"] else (n_pages, page, hk, d)
    s.k_pool, s.v_pool = (_randn(shape, gen, kind) for _ in range(2))
    s.k_pages, s.v_pages = (p.transpose(1, 2) if c["heads_first"] else p for p in (s.k_pool, s.v_pool))  # [pages, page, heads, d]
    order = random.Random(int(seed)).sample(range(n_pages), n_pages)
    table, at, starts = torch.zeros((len(s.lens), widest), dtype=torch.int32), 0, [0]
    for i, (n, _) in enumerate(s.lens):
        table[i, :held[i]] = torch.tensor(order[at:at + held[i]], dtype=torch.int32)
        at += held[i]
        starts.append(starts[-1] + n)
    s.table = table.cuda()
    s.row_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s.kv_len = torch.tensor([k for _, k in s.lens], dtype=torch.int32, device="cuda")
    # for each row of the batch its sequence and position
    s.row_seq = torch.tensor([i for i, (n, _) in enumerate(s.lens) for _ in range(n)], device="cuda")
    s.row_pos = torch.tensor([k - n + j for n, k in s.lens for j in range(n)], device="cuda")
    if c["kind"] == "append":
        s.qkv = _randn((s.rows, (hq + 2 * hk) * d), gen, TYPES[c["source"]], 1.5)
        s.q_weight, s.k_weight = (1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen) for _ in range(2))
        half = c["rope_dims"] // 2
        s.freq = c["theta"] ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(half, 1))
        s.q_out = torch.empty((s.rows, hq, d), dtype=kind, device="cuda")
    else:
        s.q = _randn((s.rows, hq, d), gen, kind, c["sharp"])
        s.sinks = torch.randn(hq, device="cuda", generator=gen) if c["sinks"] else None
        s.out = torch.empty_like(s.q)
        # the sequences that bring equally many rows, and those rows
        s.groups = []
        for n in sorted({n for n, _ in s.lens if n}):
            seqs = [i for i, (m, _) in enumerate(s.lens) if m == n]
            rows = torch.tensor([[starts[i] + j for j in range(n)] for i in seqs], device="cuda")
            s.groups.append((torch.tensor(seqs, device="cuda"), rows, max(s.lens[i][1] for i in seqs)))
    if own:
        _bind(s)  # the handle that a program of this framework keeps
    return s


class _Program:
    """What a program of this framework has for its whole life, whatever its inputs: one backend, and layers that are installed in it."""
    backend, layers = None, 0

    @classmethod
    def new_layer(cls):
        """The backend, and a layer of it that no state in use has: a layer's constants are a state's own, as its inputs are."""
        import mer_b200
        if cls.backend is None:
            cls.backend = mer_b200.Backend(mer_b200.DTYPE_Q8_0, 64, 64, 1 << 20, 1, max_tokens=1, max_top_k=1)
        cls.layers += 1
        return cls.backend, cls.layers % 64


def _bind(s):
    import mer_b200
    c, host = s.case, lambda t: None if t is None else t.cpu().numpy()
    types = {"f32": mer_b200.VALUE_F32, "f16": mer_b200.VALUE_F16, "bf16": mer_b200.VALUE_BF16}
    s.backend, s.layer = _Program.new_layer()
    append = c["kind"] == "append"
    more = dict(q_norm=host(s.q_weight) if c["norm"] else None, k_norm=host(s.k_weight) if c["norm"] else None, norm_eps=EPS, rope_freq=host(s.freq),
                rope_pairs=c["pairs"]) if append else dict(window=c["window"], sinks=host(s.sinks))
    s.backend.install_attention(s.layer, c["q_heads"], c["kv_heads"], c["head_dim"], types[c["cache"]], c["page"], **more)
    s.batch = mer_b200.KvBatch(k_pages=s.k_pages.data_ptr(), v_pages=s.v_pages.data_ptr(), n_pages=s.k_pages.shape[0], page_stride=s.k_pages.stride(0),
                               token_stride=s.k_pages.stride(1), head_stride=s.k_pages.stride(2), page_table=s.table.data_ptr(),
                               table_stride=s.table.shape[1], row_start=s.row_start.data_ptr(), kv_len=s.kv_len.data_ptr(), n_seqs=len(s.lens), n_rows=s.rows)
    if append:
        q, k, v = _parts(s)
        s.qkv_rows = mer_b200.QkvRows(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=s.q_out.data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0),
                                      v_stride=v.stride(0), value_type=types[c["source"]])


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    s = state
    append = s.case["kind"] == "append"
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if append:
            s.backend.kv_append_device(s.layer, s.batch, s.qkv_rows, stream)
        else:
            s.backend.attention_forward_device(s.layer, s.batch, s.q.data_ptr(), s.out.data_ptr(), stream)
    elif append:
        _append(s)
    else:
        _attend(s)
    return {"q": s.q_out, "k_cache": s.k_pool, "v_cache": s.v_pool} if append else {"out": s.out}


def _parts(s):
    """Queries, keys and values of the rows: parts of one matrix."""
    c = s.case
    q, k = c["q_heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    x = s.qkv
    return x[:, :q].view(s.rows, -1, c["head_dim"]), x[:, q:q + k].view(s.rows, -1, c["head_dim"]), x[:, q + k:].view(s.rows, -1, c["head_dim"])


def _append(s):
    c = s.case
    q, k, v = (x.float() for x in _parts(s))
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(2, keepdim=True) + EPS) * s.q_weight
        k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * s.k_weight
    angle = (s.row_pos.double()[:, None] * s.freq)[:, None]  # 64 bits: a far position times a frequency
    cos, sin = angle.cos().float(), angle.sin().float()
    q, k = _rotated(q, cos, sin, c), _rotated(k, cos, sin, c)
    s.q_out.copy_(q)
    page = s.table[s.row_seq, s.row_pos // c["page"]].long()
    slot = s.row_pos % c["page"]
    s.k_pages[page, slot] = k.to(s.k_pool.dtype)
    s.v_pages[page, slot] = v.to(s.v_pool.dtype)


def _rotated(x, cos, sin, c):
    r = c["rope_dims"]
    if r == 0:
        return x
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["pairs"] else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), 3).flatten(2) if c["pairs"] else torch.cat((a, b), 2)
    return torch.cat((turned, x[..., r:]), 2)


def _attend(s):
    c = s.case
    hk, d, page = c["kv_heads"], c["head_dim"], c["page"]
    for seqs, rows, longest in s.groups:  # one of them, or two where a chunk and single tokens share a step, or a prompt each
        at = torch.arange(longest, device="cuda")
        pages, slots = s.table[seqs][:, at // page].long(), at % page
        k, v = s.k_pages[pages, slots].float(), s.v_pages[pages, slots].float()  # [sequences, tokens, heads, d]
        n, m = rows.shape
        q = s.q[rows].float().view(n, m, hk, -1, d).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
        scores = (q @ k.permute(0, 2, 3, 1)).view(n, hk, m, -1, longest).mul_(d ** -0.5)
        pos = s.row_pos[rows][:, None, :, None, None]
        hidden = at > pos
        if c["window"]:
            hidden = hidden | (at <= pos - c["window"])
        scores.masked_fill_(hidden, -math.inf)
        top = scores.amax(4, keepdim=True)
        if s.sinks is not None:
            sink = s.sinks.view(1, hk, 1, -1, 1)
            top = torch.maximum(top, sink)
        scores = scores.sub_(top).exp_()
        total = scores.sum(4, keepdim=True)
        if s.sinks is not None:
            total = total + (sink - top).exp()
        o = (scores.view(n, hk, -1, longest) @ v.permute(0, 2, 1, 3)).view(n, hk, m, -1, d) / total
        s.out[rows] = o.permute(0, 2, 1, 3, 4).reshape(n, m, -1, d).to(s.out.dtype)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s, c = prepare(case, seed), case
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    f64 = torch.float64
    if c["kind"] == "append":
        x = s.qkv.to(f64).view(s.rows, hq + 2 * hk, d)
        gain = torch.ones((hq + 2 * hk, d), dtype=f64, device="cuda")
        if c["norm"]:
            gain[:hq], gain[hq:hq + hk] = s.q_weight.to(f64), s.k_weight.to(f64)
            size = (x.pow(2).sum(2, keepdim=True) / d + EPS).sqrt()
            size[:, hq + hk:] = 1.0
            x = x / size * gain
        # a rotation is a product with a complex number
        r = c["rope_dims"]
        if r:
            turn = torch.polar(torch.ones((s.rows, r // 2), dtype=f64, device="cuda"), s.row_pos.to(f64)[:, None] * s.freq)[:, None]
            first, second = (slice(0, r, 2), slice(1, r, 2)) if c["pairs"] else (slice(0, r // 2), slice(r // 2, r))
            z = torch.complex(x[:, :hq + hk, first], x[:, :hq + hk, second]) * turn
            x = x.clone()
            x[:, :hq + hk, first], x[:, :hq + hk, second] = z.real, z.imag
        pools = []
        for pool, heads in ((s.k_pool, x[:, hq:hq + hk]), (s.v_pool, x[:, hq + hk:])):
            pool = pool.to(f64)
            pages = pool.transpose(1, 2) if c["heads_first"] else pool
            for i, (n, k) in enumerate(s.lens):
                rows, at = range(int(s.row_start[i]), int(s.row_start[i + 1])), torch.arange(k - n, k, device="cuda")
                if n:
                    pages[s.table[i, at // page].long(), at % page] = heads[rows.start:rows.stop]
            pools.append(pool)
        return {"q": x[:, :hq].contiguous(), "k_cache": pools[0], "v_cache": pools[1]}
    out = torch.zeros((s.rows, hq, d), dtype=f64, device="cuda")
    g = hq // hk
    for i, (n, k) in enumerate(s.lens):
        row0 = int(s.row_start[i])
        last = max(0, k - n - c["window"] + 1) if c["window"] else 0  # the first token that any row sees
        at = torch.arange(last, k, device="cuda")
        pages = s.table[i, at // page].long()
        for h in range(hk if n else 0):
            keys, values = s.k_pages[pages, at % page, h].to(f64), s.v_pages[pages, at % page, h].to(f64)
            for j0 in range(0, n, 1024):  # rows at a time
                j1 = min(n, j0 + 1024)
                q = s.q[row0 + j0:row0 + j1, h * g:(h + 1) * g].to(f64)
                score = torch.einsum("jgd,td->jgt", q, keys) / math.sqrt(d)
                pos = torch.arange(k - n + j0, k - n + j1, device="cuda")[:, None, None]
                seen = (at <= pos) & (at > pos - c["window"]) if c["window"] else at <= pos
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                log_sum = torch.logsumexp(score, 2, keepdim=True)
                if s.sinks is not None:
                    log_sum = torch.logaddexp(log_sum, s.sinks.to(f64)[h * g:(h + 1) * g].view(1, g, 1))
                out[row0 + j0:row0 + j1, h * g:(h + 1) * g] = torch.einsum("jgt,td->jgd", (score - log_sum).exp(), values)
    return {"out": out}
