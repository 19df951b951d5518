// How the attention kernels cut a batch into equal runs of work: plain arithmetic, for the device and for the host's tests.
#pragma once

#include <stdint.h>

#include "attention.h"

#ifdef __CUDACC__
#define ATTEND_HD __host__ __device__ __forceinline__
#else
#define ATTEND_HD inline
#endif

ATTEND_HD uint32_t divided(uint32_t n, const FastDiv &f) { return ((uint32_t)((uint64_t)n * f.mul >> 32) + n) >> f.shift; }
// 64-bit division is 70 instructions; nearly always 32 bits will do.
ATTEND_HD uint64_t divided(uint64_t a, uint64_t b) { return ((a | b) >> 32) == 0 ? (uint64_t)((uint32_t)a / (uint32_t)b) : a / b; }

// Sum over 0 <= i < n of floor((a i + b) / m), a n + b below 2^32: points of the grid under a line, n columns of them.  Whole steps of slope and start
// apart, the last column is `top` high and holds the most; of the n * top points up to there, row j + 1 has those of its columns above the line that start before the
// line reaches it, ceil((m (j + 1) - b) / a): a sum of the same kind with a and m in each other's places, to be taken away.  As many turns as Euclid's algorithm has.
ATTEND_HD uint64_t points_under(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  uint64_t sum = 0;
  for (bool away = false; n; away = !away) {
    uint64_t part = (uint64_t)n * (n - 1) / 2 * (a / m) + (uint64_t)n * (b / m);
    a %= m, b %= m;
    const uint32_t top = (a * (n - 1) + b) / m, slope = a;
    part += (uint64_t)n * top;
    sum = away ? sum - part : sum + part;
    n = top, b = m - b + slope - 1, a = m, m = slope;
  }
  return sum;
}

// One sequence as a kernel with tiles of `tokens` tokens sees it.
struct SeqWork {
  uint32_t row0;    // the batch's row of its first token that has a place in the sequence
  uint32_t n, past; // such tokens, and those of the cache before them
  uint32_t tiles;   // per head

  // Blocks of the first `j` tiles of a head.
  template <uint32_t KB>
  ATTEND_HD uint64_t blocks_before(uint32_t j, uint32_t tokens, uint32_t window) const {
    if (j == 0) return 0;
    if (tiles == 1) {
      uint32_t lo, hi;
      tile_blocks<KB>(0, tokens, window, &lo, &hi);
      return hi - lo;
    }
    const uint32_t full = j == tiles ? j - 1 : j;  // the last tile may be a short one
    uint64_t hi = full == 0 ? 0 : points_under(full, KB, tokens, past + tokens + KB - 1);
    if (full != j) hi += (past + n + KB - 1) / KB;
    if (window == 0) return hi;
    // a tile's first row sees nothing before past + j * tokens - window + 1
    const uint32_t from = past + 1 >= window ? 0 : (window - 1 - past + tokens - 1) / tokens;
    return from >= j ? hi : hi - points_under(j - from, KB, tokens, past + from * tokens + 1 - window);
  }
  template <uint32_t KB>
  ATTEND_HD void tile_blocks(uint32_t j, uint32_t tokens, uint32_t window, uint32_t *lo, uint32_t *hi) const {
    const uint32_t first = j * tokens, last = (first + tokens < n ? first + tokens : n);
    *hi = (past + last + KB - 1) / KB;
    *lo = window && past + first + 1 > window ? (past + first + 1 - window) / KB : 0u;
  }
};

// How heads and rows of a layer lie in tiles of R rows: heads of a group are taken `heads` at a time.
struct TileShape {
  uint32_t group, chunks, heads, tokens, v_heads;
  uint32_t start, dense, sparse_rows, whole;  // sparse_rows: a sequence with more has dense blocks; whole: blocks of a tile that is not cut
  TileShape(uint32_t q_heads, uint32_t kv_heads, uint32_t R, uint32_t start_, uint32_t dense_, uint32_t sparse_rows_, uint32_t whole_)
      : start(start_), dense(dense_), sparse_rows(sparse_rows_), whole(whole_) {
    group = q_heads / kv_heads;
    chunks = (group + R - 1) / R;
    heads = (group + chunks - 1) / chunks;
    chunks = (group + heads - 1) / heads;
    tokens = R / heads;
    v_heads = kv_heads * chunks;
  }
};

// Units of a block of a sequence.
ATTEND_HD uint32_t block_units(const TileShape &ts, uint32_t n) { return n * ts.heads > ts.sparse_rows ? ts.dense : 1; }

// The cut of a batch's units into runs of `each` or one more: the first `more` of them have one more.
struct RunCut {
  uint64_t total, each;
  uint32_t parts, more;  // CTAs that share the work
};
ATTEND_HD RunCut cut_runs(uint64_t total, uint32_t ctas, uint32_t min_units) {
  const uint64_t most = min_units == 1 ? total : divided(total, (uint64_t)min_units);
  RunCut r;
  r.total = total;
  r.parts = most < 1 ? 1 : most < ctas ? (uint32_t)most : ctas;
  r.each = divided(total, (uint64_t)r.parts);
  r.more = (uint32_t)(total - r.each * r.parts);
  return r;
}
// First unit of a CTA's run.
ATTEND_HD uint64_t run_first(const RunCut &r, uint32_t cta) { return r.each * cta + (cta < r.more ? cta : r.more); }
// The CTA whose run holds unit x.
ATTEND_HD uint32_t run_of(const RunCut &r, uint64_t x) {
  const uint64_t wide = (r.each + 1) * r.more;
  return x < wide ? (uint32_t)divided(x, r.each + 1) : r.more + (uint32_t)divided(x - wide, r.each);
}

// A tile's part in a run.
struct TileCut {
  uint64_t at;               // the unit of the tile's first block among all
  uint32_t units;            // of a block
  uint32_t lo, hi;           // blocks of this run, none where they are equal
  uint32_t tile_lo, tile_hi; // blocks of the whole tile
};
// The part of a tile from its unit `from` on, which is unit `at` of all, for a run with `left` units to go; the units it takes.  A block is the run's that its first
// unit lies in; a tile of few blocks is wholly the run's that its own first unit lies in: joining parts of it would take longer than its blocks.
ATTEND_HD uint32_t cut_tile(const TileShape &ts, uint32_t n, uint64_t at, uint32_t from, uint64_t left, TileCut *t) {
  t->units = block_units(ts, n);
  const uint32_t all = ts.start + (t->tile_hi - t->tile_lo) * t->units, to = all < from + left ? all : (uint32_t)(from + left);
  const auto blocks_until = [&](uint32_t unit) { return unit <= ts.start ? 0u : t->units == 1 ? unit - ts.start : (unit - ts.start + t->units - 1) / t->units; };
  t->at = at - from + ts.start;
  if (t->tile_hi - t->tile_lo <= ts.whole)
    t->lo = t->tile_lo, t->hi = from == 0 ? t->tile_hi : t->tile_lo;
  else
    t->lo = t->tile_lo + blocks_until(from), t->hi = t->tile_lo + blocks_until(to);
  return to - from;
}
// The runs that have a part of a tile: c0, and n - 1 after it.
ATTEND_HD void runs_of_tile(const RunCut &run, const TileCut &t, uint32_t *c0, uint32_t *n) {
  *c0 = run_of(run, t.at);
  *n = run_of(run, t.at + (uint64_t)(t.tile_hi - t.tile_lo - 1) * t.units) - *c0 + 1;
}
// Where a CTA leaves its part of a tile: a run has parts of two tiles at most, its first and its last.
ATTEND_HD uint32_t part_slot(const RunCut &r, const TileCut &t, uint32_t cta) { return 2 * cta + (run_first(r, cta) >= t.at ? 0 : 1); }
// The same for part k of a tile that run c0 begins.
ATTEND_HD uint32_t slot_of_part(const RunCut &r, const TileCut &t, uint32_t c0, uint32_t k) { return k == 0 ? part_slot(r, t, c0) : 2 * (c0 + k); }
