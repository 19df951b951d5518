"""Host side of the attention kernels, without a GPU: how a batch is cut into runs, the pages' tensor maps, the divisions, the
refusals that need no device."""
import ctypes as C
import os
import random
import subprocess

import pytest

import mer_b200

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "micro-expert-router-ssd-streamed-moe-mer_b200", "csrc")

SOURCE = r"""
#include <cuda_runtime.h>
#include "attend_work.h"
#include "page_map.h"
extern "C" {
uint32_t div_by(uint32_t n, uint32_t d) { return divided(n, fast_div(d)); }
void shape(uint32_t q_heads, uint32_t kv_heads, uint32_t rows, uint32_t *out) {
  const TileShape t(q_heads, kv_heads, rows, 0, 1, 0, 0);
  out[0] = t.group, out[1] = t.chunks, out[2] = t.heads, out[3] = t.tokens, out[4] = t.v_heads;
}
uint64_t before(uint32_t past, uint32_t n, uint32_t tokens, uint32_t j, uint32_t window) {
  SeqWork w{0, n, past, (n + tokens - 1) / tokens};
  return w.blocks_before<128>(j, tokens, window);
}
void blocks(uint32_t past, uint32_t n, uint32_t tokens, uint32_t j, uint32_t window, uint32_t *lo, uint32_t *hi) {
  SeqWork w{0, n, past, (n + tokens - 1) / tokens};
  w.tile_blocks<128>(j, tokens, window, lo, hi);
}
// tiles: [n][3] rows of the tile's sequence, its first block, the block behind its last.  cuts: [ctas][most][4] tile, first block, block behind the last, slot (~0: whole)
uint32_t cut(const uint32_t *tiles, uint32_t n, uint32_t heads, uint32_t start, uint32_t dense, uint32_t sparse, uint32_t whole, uint32_t ctas, uint32_t min_units, uint32_t most, uint32_t *cuts,
             uint32_t *owners) {
  TileShape ts(heads, 1, 256, start, dense, sparse, whole);
  uint64_t total = 0;
  for (uint32_t i = 0; i < n; i++) total += start + (uint64_t)(tiles[3 * i + 2] - tiles[3 * i + 1]) * block_units(ts, tiles[3 * i]);
  const RunCut r = cut_runs(total, ctas, min_units);
  for (uint32_t c = 0; c < r.parts; c++) {
    uint64_t at = run_first(r, c), left = run_first(r, c + 1) - at, first = 0;
    uint32_t i = 0, k = 0;
    for (;; i++) {
      const uint64_t all = start + (uint64_t)(tiles[3 * i + 2] - tiles[3 * i + 1]) * block_units(ts, tiles[3 * i]);
      if (at < first + all) break;
      first += all;
    }
    for (uint32_t from = (uint32_t)(at - first); left; from = 0, i++) {
      TileCut t;
      t.tile_lo = tiles[3 * i + 1], t.tile_hi = tiles[3 * i + 2];
      const uint32_t taken = cut_tile(ts, tiles[3 * i], at, from, left, &t);
      at += taken, left -= taken;
      if (t.lo >= t.hi) continue;
      if (k == most) return 0;
      uint32_t *o = cuts + ((size_t)c * most + k++) * 4;
      o[0] = i + 1, o[1] = t.lo, o[2] = t.hi, o[3] = t.lo == t.tile_lo && t.hi == t.tile_hi ? 0xFFFFFFFFu : part_slot(r, t, c);
      uint32_t c0 = c, parts = 1;
      if (o[3] != 0xFFFFFFFFu) runs_of_tile(r, t, &c0, &parts);
      owners[2 * i] = c0, owners[2 * i + 1] = parts;
      if (o[3] != 0xFFFFFFFFu && slot_of_part(r, t, c0, c - c0) != o[3]) return 0;
    }
  }
  return r.parts;
}
uint32_t page_map(uint32_t kv_heads, uint32_t head_dim, uint32_t page_tokens, uint64_t page, uint64_t token, uint64_t head, uint32_t n_pages, uint32_t most, uint64_t *dims,
                  uint64_t *strides, uint32_t *box) {
  AttnLayer a{};
  KvBatchDev kv{};
  a.kv_heads = kv_heads, a.head_dim = head_dim, a.page_tokens = page_tokens;
  kv.page_stride = page, kv.token_stride = token, kv.head_stride = head, kv.n_pages = n_pages;
  const PageMapShape m(a, kv, most);
  for (int i = 0; i < 4; i++) dims[i] = m.dims[i], box[i] = m.box[i];
  for (int i = 0; i < 3; i++) strides[i] = m.strides[i];
  return m.rows | (m.head_first ? 0x10000u : 0u);
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("attend")
    src, lib = d / "rules.cpp", d / "librules.so"
    src.write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-I", "/usr/local/cuda/include", str(src), "-o", str(lib)])
    r = C.CDLL(str(lib))
    r.before.restype = C.c_uint64
    r.page_map.argtypes = [C.c_uint32] * 3 + [C.c_uint64] * 3 + [C.c_uint32] * 2 + [C.c_void_p] * 3
    return r


def test_division_by_any_page_size(rules):
    rng = random.Random(0)
    for d in [*range(1, 300), 1 << 19, (1 << 20) - 1, 1 << 20, *(rng.randrange(1, 1 << 20) for _ in range(300))]:
        for n in {0, d - 1, d, d + 1, 7 * d - 1, 2 ** 31 - 1, *(rng.randrange(1 << 31) for _ in range(8))}:
            assert rules.div_by(n, d) == n // d, (n, d)


@pytest.mark.parametrize("rows", [16, 128, 256])
def test_heads_and_tokens_of_a_tile(rules, rows):
    out = (C.c_uint32 * 5)()
    for kv in (1, 2, 8):
        for group in [*range(1, 70), 255, 256, 257, 1000]:
            rules.shape(kv * group, kv, rows, out)
            g, chunks, heads, tokens, v_heads = out
            assert g == group and v_heads == kv * chunks and 1 <= tokens and tokens * heads <= rows
            assert (chunks - 1) * heads < group <= chunks * heads  # every chunk has a head


def tile(past, n, j, tokens, window):
    first, last = past + j * tokens, past + min(n, (j + 1) * tokens)
    return max(0, first - window + 1) // 128 if window else 0, -(-last // 128)


def test_blocks_of_tiles_are_summed_in_closed_form(rules):
    rng = random.Random(1)
    lo, hi = C.c_uint32(), C.c_uint32()
    for _ in range(1500):
        tokens, n = rng.choice([1, 2, 3, 5, 16, 25, 32, 51, 64, 128, 256]), rng.randint(1, rng.choice([1, 6, 300, 4000]))
        past, window = rng.choice([0, rng.randint(0, 60), rng.randint(0, 6000)]), rng.choice([0, 0, 1, 2, 128, rng.randint(1, 7000)])
        total, tiles = 0, -(-n // tokens)
        at = {rng.randrange(tiles + 1) for _ in range(6)} | {tiles}
        for j in range(tiles + 1):
            if j in at:
                assert rules.before(past, n, tokens, j, window) == total
            if j < tiles:
                rules.blocks(past, n, tokens, j, window, C.byref(lo), C.byref(hi))
                assert (lo.value, hi.value) == tile(past, n, j, tokens, window) and lo.value < hi.value
                total += hi.value - lo.value
    # two thousand million tokens
    assert rules.before(2 ** 31 - 70000, 4096, 32, 128, 0) == sum(tile(2 ** 31 - 70000, 4096, j, 32, 0)[1] for j in range(128))


@pytest.mark.parametrize("start,dense,sparse,whole,min_units", [(3, 1, 0, 4, 1), (4, 2, 128, 6, 4), (0, 1, 0, 0, 1), (1, 2, 64, 1, 2)])
def test_runs_have_every_block_once_and_the_parts_where_the_join_looks(rules, start, dense, sparse, whole, min_units):
    rng = random.Random(start)
    for ctas in (1, 2, 7, 148):
        for _ in range(60):
            heads, tiles = rng.choice([1, 4, 8]), []
            for _ in range(rng.randint(1, 40)):
                n, lo = rng.choice([1, 1, 5, 40, 700]), rng.choice([0, 0, 3])
                tiles.append((n, lo, lo + rng.randint(1, rng.choice([1, 4, 60, 400]))))
            flat, most = [v for t in tiles for v in t], len(tiles) + 2
            cuts, owners = (C.c_uint32 * (ctas * most * 4))(), (C.c_uint32 * (2 * len(tiles)))()
            parts = rules.cut((C.c_uint32 * len(flat))(*flat), len(tiles), heads, start, dense, sparse, whole, ctas, min_units, most, cuts, owners)
            assert 1 <= parts <= ctas
            got, slots = {}, set()
            for c in range(parts):
                for k in range(most):
                    i, lo, hi, slot = cuts[(c * most + k) * 4:(c * most + k) * 4 + 4]
                    if i:
                        got.setdefault(i - 1, []).append((c, lo, hi))
                        if slot != 0xFFFFFFFF:
                            assert slot // 2 == c and slot not in slots
                            slots.add(slot)
            for i, (n, lo, hi) in enumerate(tiles):
                assert got[i][0][1] == lo and got[i][-1][2] == hi and all(a[2] == b[1] for a, b in zip(got[i], got[i][1:]))
                assert hi - lo > whole or len(got[i]) == 1
                assert [c for c, _, _ in got[i]] == list(range(owners[2 * i], owners[2 * i] + owners[2 * i + 1]))


def test_pages_have_maps_of_the_documented_kind_or_none(rules):
    dims, strides, box = (C.c_uint64 * 4)(), (C.c_uint64 * 3)(), (C.c_uint32 * 4)()
    for heads in (1, 2, 8):
        for d in (8, 64, 80, 128, 256):
            for page in (1, 3, 8, 16, 24, 40, 48, 128, 200, 256):
                for most in (16, 128):
                    for token, head, stride in ((heads * d, d, page * heads * d), (d, page * d, page * heads * d), (heads * d, d, 2 * page * heads * d),
                                                (heads * d, d, page * heads * d + 8), (d + 8, (d + 8) * page, (d + 8) * page * heads),
                                                (d, page * d * 50, page * d)):
                        got = rules.page_map(heads, d, page, stride, token, head, 50, most, dims, strides, box)
                        rows, head_first = got & 0xFFFF, got >> 16
                        if rows == 0:
                            continue
                        assert rows % 8 == 0 and page % rows == 0 and most % rows == 0  # whole swizzle atoms that stay in their page and block
                        assert list(dims) == [d, *((heads, page) if head_first else (page, heads)), 50]
                        assert list(box) == [64, *((1, rows) if head_first else (rows, 1)), 1] and box[0] * 2 == 128
                        assert all(s % 16 == 0 and s < 2 ** 40 for s in strides)
                        assert strides[0] >= 2 * d and all(strides[i] >= strides[i - 1] * dims[i] and strides[i] % strides[i - 1] == 0 for i in (1, 2))
                        # a value lies where the map looks for it
                        for p, t, h in ((0, 0, 0), (49, page - 1, heads - 1), (7, page // 2, 0)):
                            one, two = (h, t) if head_first else (t, h)
                            assert one * strides[0] + two * strides[1] + p * strides[2] == 2 * (p * stride + t * token + h * head)
    # whole pages of 16 in the usual order have one, pages of 5 have none, and neither have heads that lie outside of the pages
    assert rules.page_map(4, 128, 16, 16 * 512, 512, 128, 9, 128, dims, strides, box) & 0xFFFF == 16
    assert rules.page_map(4, 128, 256, 256 * 512, 512, 128, 9, 128, dims, strides, box) & 0xFFFF == 128
    assert rules.page_map(4, 128, 5, 5 * 512, 512, 128, 9, 128, dims, strides, box) & 0xFFFF == 0
    assert rules.page_map(4, 128, 16, 16 * 128, 128, 16 * 128 * 9, 9, 128, dims, strides, box) & 0xFFFF == 0


def test_calls_without_a_backend_are_refused():
    lib = mer_b200.load_library()
    batch, rows = mer_b200.KvBatch(), mer_b200.QkvRows()
    assert lib.mer_attention_install(None, 0, None) == 12
    assert lib.mer_kv_append_device(None, 0, batch, rows, None) == 12
    assert lib.mer_attention_forward_device(None, 0, batch, None, 0, None, 0, None) == 12


def test_the_mirror_has_the_headers_layout(tmp_path):
    capi = __import__("importlib").import_module("mer_b200.capi")
    names = {"mer_attention_cfg": capi.MerAttentionCfg, "mer_kv_batch": mer_b200.KvBatch, "mer_qkv_rows": mer_b200.QkvRows}
    body = "".join(f'printf("{s} %zu", sizeof({s}));' + "".join(f'printf(" %zu", offsetof({s}, {f[0]}));' for f in t._fields_) + 'printf("\\n");' for s, t in names.items())
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include "mer_b200.h"\nint main(void) {' + body + "return 0; }\n")
    subprocess.check_call(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    for line in subprocess.check_output([str(exe)], text=True).splitlines():
        s, size, *offsets = line.split()
        assert int(size) == C.sizeof(names[s]) and [int(o) for o in offsets] == [getattr(names[s], f[0]).offset for f in names[s]._fields_]
