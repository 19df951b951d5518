// What the attention kernels share: how the work of a batch is cut into equal parts, and how the parts of a tile are joined.
//
// A tile is up to R rows (tokens x the query heads of one key head) of one sequence; its work is counted in blocks of KB tokens
// of the cache, of which it has only those that one of its rows sees.  The blocks of all tiles in order
// (sequence, key head, tile) are cut into one equal run per CTA, so a long sequence is split over many CTAs and many short ones
// share one, whatever the lengths are; nothing of this needs the lengths on the host.  A tile that lies in the runs of several CTAs is
// joined by the one that arrives last, in the order of the runs: results do not depend on who that is.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "attention.h"
#include "../../include/mer_b200.h"

namespace {

// sum over 0 <= i < n of floor((a i + b) / m), a, b >= 0: the lattice points under a line, by Euclid's steps on (a, m).
__device__ __forceinline__ uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
  uint64_t sum = 0;
  while (n) {
    if (a >= m) sum += (n - 1) * n / 2 * (a / m), a %= m;
    if (b >= m) sum += n * (b / m), b %= m;
    const uint64_t y = a * n + b;
    if (y < m) break;
    n = y / m, b = y % m;
    const uint64_t t = m;
    m = a, a = t;
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
  __device__ __forceinline__ uint64_t blocks_before(uint32_t j, uint32_t tokens, uint32_t window) const {
    if (j == 0) return 0;
    const uint32_t full = j == tiles ? j - 1 : j;  // the last tile may be a short one
    uint64_t hi = full == 0 ? 0 : floor_sum(full, KB, tokens, (uint64_t)past + tokens + KB - 1);
    if (full != j) hi += ((uint64_t)past + n + KB - 1) / KB;
    if (window == 0) return hi;
    // a tile's first row sees nothing before past + j * tokens - window + 1
    const uint32_t from = past + 1 >= window ? 0 : (window - 1 - past + tokens - 1) / tokens;
    return from >= j ? hi : hi - floor_sum(j - from, KB, tokens, (uint64_t)past + (uint64_t)from * tokens + 1 - window);
  }
  template <uint32_t KB>
  __device__ __forceinline__ void tile_blocks(uint32_t j, uint32_t tokens, uint32_t window, uint32_t *lo, uint32_t *hi) const {
    const uint64_t first = (uint64_t)j * tokens, last = min((uint64_t)n, first + tokens);
    *hi = (uint32_t)((past + last + KB - 1) / KB);
    *lo = window && past + first + 1 > window ? (uint32_t)((past + first + 1 - window) / KB) : 0u;
  }
};

// How heads and rows of a layer lie in tiles of R rows: heads of a group are taken `heads` at a time.
struct TileShape {
  uint32_t group, chunks, heads, tokens, v_heads;
  __host__ __device__ TileShape(uint32_t q_heads, uint32_t kv_heads, uint32_t R) {
    group = q_heads / kv_heads;
    chunks = (group + R - 1) / R;
    heads = (group + chunks - 1) / chunks;
    chunks = (group + heads - 1) / heads;
    tokens = R / heads;
    v_heads = kv_heads * chunks;
  }
};

// Rows of sequence s in the batch, cut to the batch: wrong tables read nothing outside it.
__device__ __forceinline__ void seq_rows(const KvBatchDev &kv, uint32_t s, uint32_t *row, uint32_t *n, uint32_t *len) {
  const uint32_t a = __ldg(kv.row_start + s), e = min(__ldg(kv.row_start + s + 1), kv.n_rows);
  *row = a;
  *n = e > a ? e - a : 0;
  *len = min(__ldg(kv.kv_len + s), 0x7FFFFFFFu);
}
// Rows that have no place (more rows than tokens) see nothing.
__device__ __forceinline__ SeqWork seq_work(const KvBatchDev &kv, uint32_t s, uint32_t tokens, uint32_t min_n, uint32_t max_n) {
  uint32_t row, n, len;
  seq_rows(kv, s, &row, &n, &len);
  if (n < min_n || n > max_n) n = 0;
  const uint32_t skip = n > len ? n - len : 0;
  SeqWork w;
  w.row0 = row + skip, w.n = n - skip, w.past = len - w.n;
  if (n == 0) w.past = 0;
  w.tiles = (w.n + tokens - 1) / tokens;
  return w;
}

// Where a CTA's run of blocks starts.
struct RunStart {
  uint64_t total;   // blocks of the batch
  uint64_t offset;  // of the run's first block in its sequence
  uint32_t seq;
  uint32_t parts;   // CTAs that share the work
};

// All threads of the CTA; `work`: 2 * THREADS / 32 + 4 words of 64 bits in shared memory.  Threads take consecutive sequences each.
template <uint32_t KB, uint32_t THREADS>
__device__ RunStart find_run(const KvBatchDev &kv, const TileShape &ts, uint32_t window, uint32_t min_n, uint32_t max_n, uint32_t cta, uint32_t ctas,
                             uint32_t min_blocks, uint64_t *work) {
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = (kv.n_seqs + THREADS - 1) / THREADS;
  const uint32_t s0 = min(kv.n_seqs, tid * each), s1 = min(kv.n_seqs, s0 + each);
  uint64_t mine = 0;
  for (uint32_t s = s0; s < s1; s++) {
    const SeqWork w = seq_work(kv, s, ts.tokens, min_n, max_n);
    mine += w.blocks_before<KB>(w.tiles, ts.tokens, window) * ts.v_heads;
  }
  uint64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint64_t o = __shfl_up_sync(0xFFFFFFFFu, incl, d);
    if (lane >= (uint32_t)d) incl += o;
  }
  if (lane == 31) work[warp] = incl;
  __syncthreads();
  uint64_t before = 0, total = 0;
  for (uint32_t i = 0; i < THREADS / 32; i++) {
    const uint64_t v = work[i];
    before += i < warp ? v : 0;
    total += v;
  }
  const uint64_t first = before + incl - mine;
  RunStart r;
  r.total = total;
  r.parts = (uint32_t)max((uint64_t)1, min((uint64_t)ctas, total / min_blocks));
  const uint64_t x0 = cta < r.parts ? total * cta / r.parts : total;
  uint64_t *found = work + THREADS / 32;
  if (tid == 0) found[0] = kv.n_seqs, found[1] = 0;
  __syncthreads();
  if (x0 >= first && x0 < first + mine) {
    uint64_t at = first;
    for (uint32_t s = s0; s < s1; s++) {
      const SeqWork w = seq_work(kv, s, ts.tokens, min_n, max_n);
      const uint64_t u = w.blocks_before<KB>(w.tiles, ts.tokens, window) * ts.v_heads;
      if (x0 < at + u) {
        found[0] = s, found[1] = x0 - at;
        break;
      }
      at += u;
    }
  }
  __syncthreads();
  r.seq = (uint32_t)found[0];
  r.offset = found[1];
  return r;
}

// The tile of a head that holds block `x` of the head's, and how many blocks the tiles before it have.  A whole warp; every lane tries a tile.
template <uint32_t KB>
__device__ __forceinline__ uint32_t find_tile(const SeqWork &w, uint32_t tokens, uint32_t window, uint64_t x, uint64_t *before) {
  uint32_t lo = 0, hi = w.tiles;  // blocks_before(lo) <= x < blocks_before(hi)
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + 31) / 32, j = min(hi, lo + step * ((threadIdx.x & 31) + 1));
    const uint32_t below = __ballot_sync(0xFFFFFFFFu, j < hi && w.blocks_before<KB>(j, tokens, window) <= x);
    const uint32_t k = __popc(below);
    hi = min(hi, lo + step * (k + 1));
    lo += step * k;
  }
  *before = w.blocks_before<KB>(lo, tokens, window);
  return lo;
}

// Which tile a CTA works on: its place in the batch and in the run.
struct TileWork {
  uint32_t row0, past;       // the sequence's first row and the tokens before it
  uint32_t token0, tokens;   // of the sequence's rows
  uint32_t kv_head, head0, heads;  // query heads head0 .. head0 + heads
  uint32_t seq, lo, hi;      // blocks of this run
  uint32_t tile_lo, tile_hi; // blocks of the whole tile
  uint64_t at;               // the tile's first block among all
};

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

// Weights of the softmax are made as 2^(s - max + P_SHIFT): an f16 then holds weights down to 2^-36 of a row's largest, so that what a
// long row's many small ones sum to is not lost.  The shift is in the sums as well and cancels.
constexpr float P_SHIFT = 12.0f;
constexpr float LOG2E = 1.4426950408889634f;

}  // namespace
