"""Performance cases of attention over a paged cache whose keys and values are held in 4 bits, measured through the package's public
entry points.

  append   the rows of a layer's fused q|k|v projection: RMSNorm of every query and key head, the position rotation, queries out, keys
           and values quantised into the pages as they are written (kv_append_device); then those rows' keys and values as the cache
           has them from now on, read back (kv_read_device)
  attend   the new rows' queries over the keys and values of their sequences in the cache (attention_forward_device)
  read     keys and values of whole sequences, as rows of numbers (kv_read_device): to hand a prefix on, or for another kernel

A group of 32 or 64 neighbouring values of a head shares a scale and a minimum, which are f16; x is held as the code
clamp(round((x - minimum) / scale), 0, 15) and stands for scale * code + minimum, where

  minimum = f16(min x),  scale = f16(f32(max x - min x) * f32(1 / 15)),  and 1 / scale is rounded to 32 bits (0 for a scale of 0).

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
MAX_SCORES = 6.8e8  # of a drawn case's plain form: the largest listed one has 6.7e8
MAX_KEYS = 2.0e8    # values of the keys that a drawn case's plain form lays out
MAX_FLOPS, MAX_BYTES = 3.0e11, 4.0e8  # of a drawn case: the longest listed one does 3.1e11
EPS = 1e-6

_BASE = dict(kind="attend", q_heads=32, kv_heads=4, head_dim=128, type="bf16", group=32, page=16, heads_first=False, pattern="decode", seqs=1,
             rows=1, idle=0, ctx_lo=0, ctx_hi=0, lens=0)
_APPEND = dict(source="bf16", norm=True, pairs=False, rope_dims=128, theta=1e6, read="bf16")
_ATTEND = dict(window=0, sinks=False, sharp=1.0)
_READ = dict(read="bf16")


def _case(**kw):
    c = {**_BASE, **{"append": _APPEND, "read": _READ}.get(kw.get("kind"), _ATTEND)}
    unknown = set(kw) - set(c) - {"name"}
    assert not unknown, unknown
    return {**c, **kw}


_MANY = dict(q_heads=32, kv_heads=4, head_dim=128)  # heads of the 128-expert layers
_FEW = dict(q_heads=32, kv_heads=8, head_dim=128)   # heads of the 8-expert layers


def listed():
    return [
        # One user's token: the smallest call there is, launch and latency.
        _case(name="append4-decode-b1", kind="append", ctx_lo=900, ctx_hi=900, **_MANY),
        # A serving batch whose projection left 32-bit rows, as the expert layers take and give them; far positions.
        _case(name="append4-decode-b64-f32", kind="append", source="f32", read="f32", seqs=64, ctx_lo=500, ctx_hi=16000, lens=1, **_MANY),
        # A prompt of 2048 tokens on its way into the cache.
        _case(name="append4-prompt-2048", kind="append", pattern="prompts", rows=2048, page=64, **_MANY),
        # Many prompts of odd lengths at once: no norms, neighbouring values rotated, half of an odd head, groups of 64, pages that are no power of two.
        _case(name="append4-ragged-d80", kind="append", type="f16", source="f16", read="f32", norm=False, pairs=True, theta=1e4, page=24, group=64, heads_first=True,
              pattern="prompts", seqs=13, rows=1333, idle=1, ctx_lo=1, ctx_hi=700, lens=2, **{**_FEW, "head_dim": 80}, rope_dims=40),
        # One user's token far into a long text: few rows, a long axis to split.
        _case(name="attend4-decode-b1-32k", ctx_lo=32000, ctx_hi=32000, **_MANY),
        # A serving batch of 64 users with contexts of very different lengths.
        _case(name="attend4-decode-b64", seqs=64, ctx_lo=800, ctx_hi=8000, lens=3, page=32, **_MANY),
        # A window of 128 tokens, a learned sink for each head, heads of 64: little to read, so latency counts.
        _case(name="attend4-decode-window-b16", q_heads=64, kv_heads=8, head_dim=64, seqs=16, ctx_lo=100, ctx_hi=4000, lens=4, window=128, sinks=True),
        # Drafts of five tokens for eight users, groups of 64.
        _case(name="attend4-draft-b8", type="f16", group=64, pattern="draft", seqs=8, rows=5, ctx_lo=1000, ctx_hi=6000, lens=5, sharp=2.0, **_FEW),
        # A chunk of a prompt and 47 users' single tokens in one step.
        _case(name="attend4-mixed-b48", pattern="mixed", seqs=48, rows=777, idle=1, ctx_lo=300, ctx_hi=6000, lens=6, page=32, sharp=2.0, **_FEW),
        # The largest call: a chunk of 2048 tokens behind 8 thousand that are in the cache.
        _case(name="attend4-chunk-2048-8k", pattern="prompts", rows=2048, ctx_lo=8200, ctx_hi=8200, page=64, **_MANY),
        # Two users' texts of some hundred tokens as 32-bit rows, in pages that no copy of sixteen tokens fits.
        _case(name="read4-short-f32", kind="read", read="f32", pattern="prompts", seqs=2, rows=300, page=24, group=64, lens=8, **_FEW),
        # A text of 32 thousand tokens as rows for another kernel.
        _case(name="read4-32k", kind="read", pattern="prompts", rows=32000, page=64, **_MANY),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kv_heads = rng.choice([1, 2, 4, 4, 8, 8])
        c = dict(kind=rng.choice(["append", "attend", "attend", "attend", "read"]), kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 8, 16]),
                 head_dim=rng.choice([64, 64, 128, 128, 128, 128, 80, 96, 256]), type=rng.choice(["bf16", "bf16", "f16"]), group=rng.choice([32, 32, 64]),
                 page=rng.choice([16, 16, 32, 64, 128, 256, 1, 24, 40]), heads_first=rng.random() < 0.3,
                 pattern=rng.choice(["decode", "decode", "draft", "prompts", "prompts", "mixed"]), idle=rng.choice([0, 0, 1, 2]), lens=rng.randrange(1 << 20))
        if c["kind"] == "read":
            c.update(pattern="prompts", read=rng.choice(["bf16", "f16", "f32"]))
        if c["pattern"] == "decode":
            c.update(seqs=_log_int(rng, 1, 200))
        elif c["pattern"] == "draft":
            c.update(seqs=_log_int(rng, 1, 48), rows=rng.randint(2, 9))
        elif c["pattern"] == "prompts":
            c.update(seqs=_log_int(rng, 1, 8), rows=_log_int(rng, 16, 32000 if c["kind"] == "read" else 4096))
        else:
            c.update(seqs=_log_int(rng, 2, 64), rows=_log_int(rng, 16, 2048))
        c["ctx_lo"] = _log_int(rng, 1, 8000) if c["kind"] != "read" and (c["pattern"] != "prompts" or rng.random() < 0.5) else 0
        c["ctx_hi"] = min(32000, c["ctx_lo"] * rng.randint(1, 10))
        if c["kind"] == "append":
            d = c["head_dim"]
            c.update(source=rng.choice(["bf16", "f32", "f16"]), norm=rng.random() < 0.6, pairs=rng.random() < 0.3, rope_dims=rng.choice([d, d, d, d // 2, 0]),
                     theta=rng.choice([1e4, 1e6, 5e5]), read=rng.choice(["bf16", "f16", "f32"]))
        elif c["kind"] == "attend":
            c.update(window=rng.choice([0, 0, 0, 128, 1024, rng.randint(1, 3000)]), sinks=rng.random() < 0.25, sharp=rng.choice([1.0, 2.0]))
        c = _case(**c)
        w, lens = work(c), lengths(c)
        scores = sum(n * k for n, k in _padded(lens)) * c["q_heads"]
        keys = sum(k for n, k in lens) * kv_heads * c["head_dim"]
        laid_out = max(s * k for s, _, k in _groups(lens)) * kv_heads * c["head_dim"]
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and keys <= MAX_KEYS and (c["kind"] != "attend" or (scores <= MAX_SCORES and laid_out <= MAX_KEYS)):
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
    held = d / 2 + 4 * -(-d // c["group"])  # bytes of a head's codes, scales and minima
    if c["kind"] == "append":
        size, out = TYPES[c["source"]].itemsize, TYPES[c["read"]].itemsize
        return {"bytes": rows * ((hq + 2 * hk) * d * size + hq * d * 2 + 2 * hk * (held + d * out)) + tables,
                "flops": rows * (hq + hk) * d * (4.0 * c["norm"] + 3.0) + rows * 2 * hk * d * 8.0}
    if c["kind"] == "read":
        return {"bytes": rows * 2 * hk * (held + d * TYPES[c["read"]].itemsize) + tables, "flops": rows * 2 * hk * d * 2.0}
    pairs = seen = 0
    for n, k in lens:
        w = c["window"] or k
        full = max(0, min(n, w - (k - n) - 1))  # rows whose window reaches before the first token
        first = k - n + 1
        pairs += full * first + full * (full - 1) // 2 + (n - full) * w if c["window"] else n * first + n * (n - 1) // 2
        seen += min(k, w + n - 1) if n else 0
    return {"bytes": rows * hq * d * 4 + seen * hk * 2 * held + tables, "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------ the cache
#
# A page of one key head is a block of bytes: the codes of its tokens one behind the other, then their scales and minima.  A head's
# codes are stored for 64, 96, 128, 192 or 256 values, `units` times 32; what is behind the head's own values is never looked at.
#
#   keys     32-bit word j * units + u of a token (j < 4) has the values 32 u + 8 j + 2 p and + 2 p + 1, from bits 4 p and 16 + 4 p on
#   values   16-bit word r * units + u of a token (r < 8) has the values 32 u + 4 r + i, from bit 4 i on
#   both     scale and minimum of group g (f16) of a token lie side by side, 4 g bytes behind those of its first group


def _units(c):
    return next(u for u in (2, 3, 4, 6, 8) if 32 * u >= c["head_dim"])


def _pack(x, c, keys):
    """(codes as words [..., words], scales and minima [..., groups, 2]) of heads [..., head_dim]."""
    u, d = _units(c), c["head_dim"]
    groups = -(-32 * u // c["group"])
    at = torch.arange(groups * c["group"], device=x.device).clamp(max=d - 1)  # the last value again: no other minimum, no other maximum
    x = x[..., at].unflatten(-1, (groups, c["group"]))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    least = lo.float().half()
    scale = ((hi - lo).float() * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).half()
    unit = torch.where(scale > 0, scale.float().reciprocal(), 0.0)
    code = ((x - least.to(x.dtype)) * unit.to(x.dtype)).round().clamp(0, 15).flatten(-2)[..., :32 * u].to(torch.int32)
    shifts = torch.arange(8, device=x.device)
    if keys:
        words = (code.unflatten(-1, (u, 4, 8)) << (shifts // 2 * 4 + shifts % 2 * 16)).sum(-1)
        words = words.transpose(-1, -2).flatten(-2).to(torch.int32)  # the sum's low 32 bits
    else:
        words = (code.unflatten(-1, (u, 8, 4)) << (shifts[:4] * 4)).sum(-1)
        words = words.transpose(-1, -2).flatten(-2).to(torch.int16)
    return words, torch.cat((scale, least), -1)


def _codes(words, c, keys):
    """The codes [..., head_dim] of words."""
    u = _units(c)
    shifts = torch.arange(8, device=words.device)
    shifts = shifts // 2 * 4 + shifts % 2 * 16 if keys else shifts[:4] * 4
    words = words.unflatten(-1, (-1, u)).transpose(-1, -2)
    return (words.to(torch.int32)[..., None] >> shifts & 15).flatten(-3)[..., :c["head_dim"]]


def _values(words, scales, c, keys):
    """The values in 32 bits that words, scales and minima stand for."""
    scale, least = scales.float().repeat_interleave(c["group"], -2)[..., :c["head_dim"], :].unbind(-1)
    return scale * _codes(words, c, keys) + least


def _parts_of(pool, c, keys):
    """Views of a pool of blocks: words [page, head, token, words], scales and minima [page, head, token, groups, 2]."""
    u = _units(c)
    size = c["page"] * 16 * u
    groups = -(-32 * u // c["group"])
    return (pool[..., :size].view(torch.int32 if keys else torch.int16).unflatten(-1, (c["page"], -1)),
            pool[..., size:size + c["page"] * 4 * groups].view(torch.float16).unflatten(-1, (c["page"], groups, 2)))


def _block_bytes(c):
    u = _units(c)
    return -(-c["page"] * (16 * u + 4 * -(-32 * u // c["group"])) // 16) * 16


# ------------------------------------------------------------------------------------------------ inputs


class _State:
    pass


def _generator(seed, tag):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + tag + 1) % (1 << 62))


def _randn(shape, gen, dtype, scale=1.0):
    return torch.randn(shape, device="cuda", generator=gen).mul_(scale).to(dtype)


def prepare(case, seed):
    c, s = case, _State()
    s.case, s.lens = c, lengths(c)
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    gen = _generator(seed, 1)
    s.rows = sum(n for n, _ in s.lens)
    # the cache: a pool of pages, of which each sequence has some in any order
    held = [-(-k // page) for _, k in s.lens]
    n_pages, widest = sum(held) + 3, max(held)
    shape = (hk, n_pages, _block_bytes(c)) if c["heads_first"] else (n_pages, hk, _block_bytes(c))
    s.pools = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s.k_pages, s.v_pages = (p.transpose(0, 1) if c["heads_first"] else p for p in s.pools)  # [page, head, bytes]
    if c["kind"] != "append":
        for pages, keys in ((s.k_pages, True), (s.v_pages, False)):
            at_once = max(1, (1 << 25) // (hk * page * d))
            for i in range(0, n_pages, at_once):
                n = min(at_once, n_pages - i)
                for to, x in zip(_parts_of(pages[i:i + n], c, keys), _pack(torch.randn((n, hk, page, d), device="cuda", generator=gen), c, keys)):
                    to.copy_(x)
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
    new = torch.tensor([n for n, _ in s.lens])
    s.row_seq = torch.repeat_interleave(torch.arange(len(s.lens)), new).cuda()
    first = torch.tensor([k - n - b for (n, k), b in zip(s.lens, starts)])
    s.row_pos = (torch.repeat_interleave(first, new) + torch.arange(s.rows)).cuda()
    if c["kind"] == "append":
        s.qkv = _randn((s.rows, (hq + 2 * hk) * d), gen, TYPES[c["source"]], 1.5)
        s.q_weight, s.k_weight = (1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen) for _ in range(2))
        half = c["rope_dims"] // 2
        s.freq = c["theta"] ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(half, 1))
        s.q_out = torch.empty((s.rows, hq, d), dtype=TYPES[c["type"]], device="cuda")
    if c["kind"] != "attend":
        s.k_out, s.v_out = (torch.empty((s.rows, hk, d), dtype=TYPES[c["read"]], device="cuda") for _ in range(2))
    else:
        s.q = _randn((s.rows, hq, d), gen, TYPES[c["type"]], c["sharp"])
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
    more = {}
    if c["kind"] == "append":
        more = dict(q_norm=host(s.q_weight) if c["norm"] else None, k_norm=host(s.k_weight) if c["norm"] else None, norm_eps=EPS, rope_freq=host(s.freq),
                    rope_pairs=c["pairs"])
    elif c["kind"] == "attend":
        more = dict(window=c["window"], sinks=host(s.sinks))
    s.backend.install_attention(s.layer, c["q_heads"], c["kv_heads"], c["head_dim"], types[c["type"]], c["page"], cache_bits=4, cache_group=c["group"], **more)
    s.batch = mer_b200.KvBatch(k_pages=s.k_pages.data_ptr(), v_pages=s.v_pages.data_ptr(), n_pages=s.k_pages.shape[0], page_stride=s.k_pages.stride(0),
                               head_stride=s.k_pages.stride(1), page_table=s.table.data_ptr(), table_stride=s.table.shape[1],
                               row_start=s.row_start.data_ptr(), kv_len=s.kv_len.data_ptr(), n_seqs=len(s.lens), n_rows=s.rows)
    if c["kind"] == "append":
        q, k, v = _parts(s)
        s.qkv_rows = mer_b200.QkvRows(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=s.q_out.data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0),
                                      v_stride=v.stride(0), value_type=types[c["source"]])
    if c["kind"] != "attend":
        s.kv_rows = mer_b200.KvRows(k=s.k_out.data_ptr(), v=s.v_out.data_ptr(), value_type=types[c["read"]])


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    s, kind = state, state.case["kind"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if kind == "append":
            s.backend.kv_append_device(s.layer, s.batch, s.qkv_rows, stream)
        if kind == "attend":
            s.backend.attention_forward_device(s.layer, s.batch, s.q.data_ptr(), s.out.data_ptr(), stream)
        else:
            s.backend.kv_read_device(s.layer, s.batch, s.kv_rows, stream)
    elif kind == "attend":
        _attend(s)
    else:
        if kind == "append":
            _append(s)
        _read(s)
    if kind == "attend":
        return {"out": s.out}
    return {"k": s.k_out, "v": s.v_out, **({"q": s.q_out} if kind == "append" else {})}


def _parts(s):
    """Queries, keys and values of the rows: parts of one matrix."""
    c = s.case
    q, k = c["q_heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    x = s.qkv
    return x[:, :q].view(s.rows, -1, c["head_dim"]), x[:, q:q + k].view(s.rows, -1, c["head_dim"]), x[:, q + k:].view(s.rows, -1, c["head_dim"])


def _place(s):
    """Page and slot of the rows."""
    return s.table[s.row_seq, s.row_pos // s.case["page"]].long(), s.row_pos % s.case["page"]


def _append(s):
    c = s.case
    q, k, v = _parts(s)
    q, k, v = q.float(), k.double(), v.double()  # 64 bits: a code next to the border between two is the nearer one's
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(2, keepdim=True) + EPS) * s.q_weight
        k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * s.k_weight
    angle = (s.row_pos.double()[:, None] * s.freq)[:, None]  # a far position times a frequency
    cos, sin = angle.cos(), angle.sin()
    q, k = _rotated(q, cos.float(), sin.float(), c), _rotated(k, cos, sin, c)
    s.q_out.copy_(q)
    page, slot = _place(s)
    for pages, x, keys in ((s.k_pages, k, True), (s.v_pages, v, False)):
        words, scales = _parts_of(pages, c, keys)
        words[page, :, slot], scales[page, :, slot] = _pack(x, c, keys)


def _rotated(x, cos, sin, c):
    r = c["rope_dims"]
    if r == 0:
        return x
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["pairs"] else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), 3).flatten(2) if c["pairs"] else torch.cat((a, b), 2)
    return torch.cat((turned, x[..., r:]), 2)


def _read(s):
    page, slot = _place(s)
    for pages, out, keys in ((s.k_pages, s.k_out, True), (s.v_pages, s.v_out, False)):
        words, scales = _parts_of(pages, s.case, keys)
        out.copy_(_values(words[page, :, slot], scales[page, :, slot], s.case, keys))


def _attend(s):
    c = s.case
    hk, d, page = c["kv_heads"], c["head_dim"], c["page"]
    for seqs, rows, longest in s.groups:  # one of them, or two where a chunk and single tokens share a step, or a prompt each
        at = torch.arange(longest, device="cuda")
        pages, slots = s.table[seqs][:, at // page].long(), at % page
        k, v = (_values(*(x[pages, :, slots] for x in _parts_of(p, c, keys)), c, keys) for p, keys in ((s.k_pages, True), (s.v_pages, False)))  # [sequences, tokens, heads, d]
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


def _held(page_bytes, c, keys, head, tokens):
    """What the cache holds for some tokens of pages [tokens, heads, block], byte by byte: [tokens, head_dim] in 64 bits."""
    u, d, g = _units(c), c["head_dim"], c["group"]
    groups = -(-32 * u // g)
    block = page_bytes[:, head]
    j = torch.arange(d, device="cuda")
    unit, inside = j // 32, j % 32
    if keys:  # which 4-bit piece of the token's codes
        piece = ((inside // 8) * u + unit) * 8 + (inside % 8) // 2 + (inside % 2) * 4
    else:
        piece = ((inside // 4) * u + unit) * 4 + inside % 4
    byte = block.gather(1, tokens[:, None] * (16 * u) + (piece // 2)[None])
    code = torch.where(piece % 2 == 1, byte // 16, byte % 16).to(torch.float64)
    first = c["page"] * 16 * u + tokens[:, None] * (4 * groups) + (j // g * 4)[None]
    def number(i):
        bits = block.gather(1, first + i).to(torch.int32) + block.gather(1, first + i + 1).to(torch.int32) * 256
        return torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16).view(torch.float16).to(torch.float64)
    return number(0) * code + number(2)


def _nearest(x, c):
    """What a 4-bit cache has in place of heads [..., head_dim] of 64-bit values."""
    got = torch.empty_like(x)
    for a in range(0, c["head_dim"], c["group"]):
        part = x[..., a:a + c["group"]]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        m = low.to(torch.float32).to(torch.float16)
        step = ((high - low).to(torch.float32) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device="cuda")).to(torch.float16)
        per = torch.where(step == 0, torch.zeros_like(step, dtype=torch.float32), 1.0 / step.to(torch.float32)).to(torch.float64)
        n = torch.floor((part - m.to(torch.float64)) * per + 0.5)
        n = n - ((n - (part - m.to(torch.float64)) * per == 0.5) & (n % 2 == 1)).to(torch.float64)  # halves go to the even one
        n = torch.minimum(torch.maximum(n, torch.zeros_like(n)), torch.full_like(n, 15.0))
        got[..., a:a + c["group"]] = n * step.to(torch.float64) + m.to(torch.float64)
    return got


def exact(case, seed):
    s, c = prepare(case, seed), case
    hq, hk, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    f64 = torch.float64
    if c["kind"] == "append":
        x = s.qkv.to(f64).view(s.rows, hq + 2 * hk, d)
        if c["norm"]:
            gain = torch.ones((hq + 2 * hk, d), dtype=f64, device="cuda")
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
        return {"q": x[:, :hq].contiguous(), "k": _nearest(x[:, hq:hq + hk], c), "v": _nearest(x[:, hq + hk:], c)}
    if c["kind"] == "read":
        got = []
        for pages, keys in ((s.k_pages, True), (s.v_pages, False)):
            out = torch.empty((s.rows, hk, d), dtype=f64, device="cuda")
            for i, (n, k) in enumerate(s.lens):
                at = torch.arange(k - n, k, device="cuda")
                for h in range(hk if n else 0):
                    out[int(s.row_start[i]):int(s.row_start[i + 1]), h] = _tokens(s, pages, keys, i, at, h)
            got.append(out)
        return {"k": got[0], "v": got[1]}
    out = torch.zeros((s.rows, hq, d), dtype=f64, device="cuda")
    g = hq // hk
    for i, (n, k) in enumerate(s.lens):
        row0 = int(s.row_start[i])
        last = max(0, k - n - c["window"] + 1) if c["window"] else 0  # the first token that any row sees
        at = torch.arange(last, k, device="cuda")
        for h in range(hk if n else 0):
            keys, values = _tokens(s, s.k_pages, True, i, at, h), _tokens(s, s.v_pages, False, i, at, h)
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


def _tokens(s, pages, keys, seq, at, head):
    """Tokens `at` of a sequence as the cache holds them, a few thousand at a time."""
    page = s.case["page"]
    return torch.cat([_held(pages[s.table[seq, a // page].long()], s.case, keys, head, a % page) for a in at.split(1024)])
