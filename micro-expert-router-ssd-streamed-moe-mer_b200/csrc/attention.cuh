// What the attention kernels share: how the work of a batch is cut into equal parts, and how the parts of a tile are joined.
//
// A tile is up to R rows (tokens x the query heads of one key head) of one sequence; its work is counted in blocks of KB tokens
// of the cache, of which it has only those that one of its rows sees.  The blocks of all tiles in order
// (sequence, key head, tile) are cut into one equal run per CTA, so a long sequence is split over many CTAs and many short ones
// share one, whatever the lengths are; nothing of this needs the lengths on the host.  The runs are equal in units: a block has one, or
// `dense` of a sequence with so many rows that its blocks take longer, and a tile has `start` units in front of its blocks, for beginning and ending it.  A tile that lies in the runs of several CTAs is
// joined by the one that arrives last, in the order of the runs: results do not depend on who that is.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "attend_work.h"
#include "attention.h"
#include "../../include/mer_b200.h"
#include "page_map.h"

namespace {

// Rows of sequence s in the batch, cut to the batch: wrong tables read nothing outside it.  Tables are read by ordinary loads: this kernel may have started
// while the one in front of it still ran, which may have written them, and loads of what is constant for a kernel's whole life are not ordered behind that.
__device__ __forceinline__ void seq_rows(const KvBatchDev &kv, uint32_t s, uint32_t *row, uint32_t *n, uint32_t *len) {
  const uint32_t a = kv.row_start[s], e = min(kv.row_start[s + 1], kv.n_rows);
  *row = a;
  *n = e > a ? e - a : 0;
  const uint32_t l = kv.kv_len[s];
  *len = l <= kv.capacity ? l : 0;  // more than the table has pages for: no row of it has a place
}
// Rows that have no place (more rows than tokens) see nothing.
__device__ __forceinline__ SeqWork seq_work(const KvBatchDev &kv, uint32_t s, uint32_t tokens) {
  uint32_t row, n, len;
  seq_rows(kv, s, &row, &n, &len);
  const uint32_t skip = n > len ? n - len : 0;
  SeqWork w;
  w.row0 = row + skip, w.n = n - skip, w.past = len - w.n;
  if (n == 0) w.past = 0;
  w.tiles = (w.n + tokens - 1) / tokens;
  return w;
}

// Where this CTA's run starts.
struct RunStart : RunCut {
  uint32_t seq;                // the sequence of the run's first unit
  uint32_t v_head, tile, from; // its head, its tile, and the tile's units before it
  SeqWork w;
};

struct RunFound {
  uint64_t sums[16], more_sums[16];
  uint64_t offset, per_head;
  SeqWork w;
  uint32_t seq, tile, from;
};

// Sum of `mine` over the threads before this one, and over all; `sums`: a word for each warp.
template <uint32_t THREADS>
__device__ __forceinline__ uint64_t scan_threads(uint64_t mine, uint64_t *sums, uint64_t *total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint64_t o = __shfl_up_sync(0xFFFFFFFFu, incl, d);
    if (lane >= (uint32_t)d) incl += o;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (uint32_t i = 0; i < THREADS / 32; i++) {
    const uint64_t v = sums[i];
    before += i < warp ? v : 0;
    all += v;
  }
  *total = all;
  return before + incl - mine;
}

// All threads of the CTA (16 warps at most), which take consecutive sequences each; `found` in shared memory.
template <uint32_t KB, uint32_t THREADS>
__device__ RunStart find_run(const KvBatchDev &kv, const TileShape &ts, uint32_t window, uint32_t cta, uint32_t ctas,
                             uint32_t min_units, RunFound &found) {
  const uint32_t tid = threadIdx.x, each = (kv.n_seqs + THREADS - 1) / THREADS;
  const uint32_t s0 = min(kv.n_seqs, tid * each), s1 = min(kv.n_seqs, s0 + each);
  uint64_t mine = 0, per_head = 0, total;
  SeqWork w{};
  for (uint32_t s = s0; s < s1; s++) {
    w = seq_work(kv, s, ts.tokens);
    per_head = w.blocks_before<KB>(w.tiles, ts.tokens, window) * block_units(ts, w.n) + w.tiles * ts.start;
    mine += per_head * ts.v_heads;
  }
  const uint64_t first = scan_threads<THREADS>(mine, found.sums, &total);
  RunStart r;
  static_cast<RunCut &>(r) = cut_runs(total, ctas, min_units);
  const uint64_t x0 = run_first(r, min(cta, r.parts));
  if (x0 >= first && x0 < first + mine) {
    uint64_t at = first;
    uint32_t s = s0;
    if (s1 - s0 > 1) {
      for (;; s++) {
        w = seq_work(kv, s, ts.tokens);
        per_head = w.blocks_before<KB>(w.tiles, ts.tokens, window) * block_units(ts, w.n) + w.tiles * ts.start;
        if (x0 < at + per_head * ts.v_heads) break;
        at += per_head * ts.v_heads;
      }
    }
    found.seq = s, found.offset = x0 - at, found.per_head = per_head, found.w = w;
  }
  if (tid == 0) found.tile = 0;
  __syncthreads();
  if (cta >= r.parts || total == 0) return r;  // no run
  r.seq = found.seq, r.w = found.w;
  r.v_head = (uint32_t)divided(found.offset, found.per_head);
  const uint64_t x = found.offset - r.v_head * found.per_head;
  if (r.w.tiles > 1) {  // threads take consecutive tiles each
    const uint32_t some = (r.w.tiles + THREADS - 1) / THREADS, j0 = min(r.w.tiles, tid * some), j1 = min(r.w.tiles, j0 + some);
    uint32_t lo, hi;
    const uint32_t units = block_units(ts, r.w.n);
    mine = 0;
    for (uint32_t j = j0; j < j1; j++) r.w.tile_blocks<KB>(j, ts.tokens, window, &lo, &hi), mine += (hi - lo) * units + ts.start;
    uint64_t at = scan_threads<THREADS>(mine, found.more_sums, &total);
    if (x >= at && x < at + mine) {
      for (uint32_t j = j0;; j++) {
        r.w.tile_blocks<KB>(j, ts.tokens, window, &lo, &hi);
        if (x < at + ((hi - lo) * units + ts.start)) {
          found.tile = j, found.from = (uint32_t)(x - at);
          break;
        }
        at += (hi - lo) * units + ts.start;
      }
    }
    __syncthreads();
    r.tile = found.tile, r.from = found.from;
  } else {
    r.tile = 0, r.from = (uint32_t)x;
  }
  return r;
}

// Where the tokens of a sequence lie, for one key head.
struct PagePlaces {
  const uint32_t *pages;
  uint32_t widest, n_pages, page_tokens, page, token, head;  // the strides in pieces of 16 bytes
  FastDiv div;

  __device__ __forceinline__ PagePlaces(const KvBatchDev &kv, uint32_t page_tokens_, uint32_t seq, uint32_t kv_head)
      : pages(kv.page_table + (uint64_t)seq * kv.table_stride), widest(kv.table_stride), n_pages(kv.n_pages), page_tokens(page_tokens_),
        page((uint32_t)(kv.page_stride / 8)), token((uint32_t)(kv.token_stride / 8)), head(kv_head * (uint32_t)(kv.head_stride / 8)), div(kv.page_tokens) {}
  // The entry of the table for a token: to be asked for well before the place.
  __device__ __forceinline__ uint32_t entry(uint32_t key) const {
    const uint32_t slot = divided(key, div);
    return slot < widest ? pages[slot] : 0xFFFFFFFFu;
  }
  __device__ __forceinline__ uint32_t in_page(uint32_t key) const { return key - divided(key, div) * page_tokens; }
  // The token's place in pieces of 16 bytes; ~0 and `bad` where the page is not there.
  __device__ __forceinline__ uint32_t place(uint32_t key, uint32_t number, uint32_t *bad) const {
    if (number >= n_pages) {
      *bad = 1;
      return 0xFFFFFFFFu;
    }
    return number * page + in_page(key) * token + head;
  }
};

// 16 bytes, of which those behind the first `bytes` are zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// 64 values of a run of tokens of a page, swizzled; zeros where the page number is not one of the map's.
__device__ __forceinline__ void page_g2s(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t token, uint32_t head, uint32_t page, bool head_first, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x),
               "r"(head_first ? head : token), "r"(head_first ? token : head), "r"(page), "r"(bar)
               : "memory");
}

// Which tile a CTA works on: its place in the batch and in the run.
struct TileWork : TileCut {
  uint32_t row0, past;             // the sequence's first row and the tokens before it
  uint32_t token0, tokens;         // of the sequence's rows
  uint32_t kv_head, head0, heads;  // query heads head0 .. head0 + heads
  uint32_t seq;
};

// The first token that a row of the tile sees.
__device__ __forceinline__ uint32_t first_seen(const TileWork &t, uint32_t window) {
  const uint32_t behind = t.past + t.token0 + 1;
  return window && behind > window ? behind - window : 0;
}

template <typename T>
struct Num;
template <>
struct Num<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ __half one(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float f(__half v) { return __half2float(v); }
};
template <>
struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ __nv_bfloat16 one(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float f(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Num<float> {
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float f(float v) { return v; }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights of the softmax are made as 2^(s - max + P_SHIFT): an f16 then holds weights down to 2^-32 of a row's largest, so that what a
// long row's many small ones sum to is not lost.  The shift is in the sums as well and cancels.
constexpr float P_SHIFT = 8.0f;
constexpr float LOG2E = 1.4426950408889634f;
// Weight of a head's sink beside scores whose reference is `top`; a sink of -infinity has none, also where all scores are -infinity.
__device__ __forceinline__ float sink_weight(const float *sinks, uint32_t head, float top) {
  const float sink = __ldg(sinks + head);
  return sink == -INFINITY ? 0.0f : exp2_approx(sink * LOG2E - top + P_SHIFT);
}

}  // namespace
