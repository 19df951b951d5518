// The way of a CTA through its run, and the end of a tile: its rows stored, or the parts of several CTAs joined.
#pragma once

#include "attention.cuh"
#include "ptx.cuh"

namespace {

template <uint32_t KB>
struct RunWalk {
  const KvBatchDev &kv;
  const TileShape &ts;
  uint32_t window;
  uint64_t left, at;  // units of the run that are left, and the next one's number
  SeqWork w;
  uint32_t seq, v_head, tile, from;  // from: what of the tile is not this run's (its first tile alone)
  bool fresh = true;

  __device__ RunWalk(const KvBatchDev &kv_, const TileShape &ts_, uint32_t window_, const RunStart &r)
      : kv(kv_), ts(ts_), window(window_), w(r.w), seq(r.seq), v_head(r.v_head), tile(r.tile), from(r.from) {
    at = run_first(r, blockIdx.x);
    left = r.total == 0 ? 0 : run_first(r, blockIdx.x + 1) - at;
  }
  // The next tile of the run, or a part of one.
  __device__ bool next(TileWork *t) {
    do {
      if (left == 0) return false;
      if (fresh) {
        fresh = false;
      } else {
        from = 0;
        if (++tile >= w.tiles) {
          tile = 0;
          if (++v_head >= ts.v_heads) {
            v_head = 0;
            do {
              seq++;
              if (seq >= kv.n_seqs) return false;
              w = seq_work(kv, seq, ts.tokens);
            } while (w.tiles == 0);
          }
        }
      }
      w.tile_blocks<KB>(tile, ts.tokens, window, &t->tile_lo, &t->tile_hi);
      const uint32_t taken = cut_tile(ts, w.n, at, from, left, t);
      left -= taken, at += taken;
    } while (t->lo >= t->hi);  // no block of it
    t->seq = seq, t->row0 = w.row0, t->past = w.past;
    t->token0 = tile * ts.tokens;
    t->tokens = min(ts.tokens, w.n - t->token0);
    t->kv_head = ts.chunks == 1 ? v_head : v_head / ts.chunks;
    const uint32_t chunk = v_head - t->kv_head * ts.chunks;
    t->head0 = t->kv_head * ts.group + chunk * ts.heads;
    t->heads = min(ts.heads, ts.group - chunk * ts.heads);
    return true;
  }
};

// Rows that have no place in their sequence (it brings more rows than it has tokens) see nothing: zero.
template <typename T, uint32_t THREADS>
__device__ void clear_rows_without_place(const AttnLayer &a, const KvBatchDev &kv, T *out, uint64_t out_stride, uint32_t *status) {
  for (uint32_t s0 = 0; s0 < kv.n_seqs; s0 += THREADS) {
    const uint32_t s = s0 + threadIdx.x;
    uint32_t row = 0, n = 0, len = 0;
    if (s < kv.n_seqs) seq_rows(kv, s, &row, &n, &len);
    const bool some = n > len;
    if (some) atomicOr(status, MER_DEVSTAT_BAD_CACHE);
    if (!__syncthreads_or(some)) continue;
    for (uint32_t i = s0; i < min(kv.n_seqs, s0 + THREADS); i++) {
      seq_rows(kv, i, &row, &n, &len);
      if (n <= len) continue;
      const uint32_t width = a.q_heads * a.head_dim;
      for (uint64_t e = threadIdx.x; e < (uint64_t)(n - len) * width; e += THREADS) out[(row + e / width) * out_stride + e % width] = Num<T>::one(0.0f);
    }
  }
}

// Floats of a part: maximum and sum of R rows, and their outputs.
__host__ __device__ constexpr uint32_t part_floats(uint32_t R, uint32_t DP) { return R * (DP + 2); }
// Four values from column c on of row r of a tile.
template <typename T>
__device__ __forceinline__ void store_row(const AttnLayer &a, const TileWork &t, uint32_t r, uint32_t c, float top, float sum, const float4 &acc, T *out, uint64_t out_stride) {
  if (c >= a.head_dim) return;
  const uint32_t tok = r / t.heads, head = t.head0 + r - tok * t.heads;
  if (a.sinks) sum += sink_weight(a.sinks, head, top);
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint2 v = make_uint2(Num<T>::pack(acc.x * f, acc.y * f), Num<T>::pack(acc.z * f, acc.w * f));
  *reinterpret_cast<uint2 *>(out + (uint64_t)(t.row0 + t.token0 + tok) * out_stride + (uint64_t)head * a.head_dim + c) = v;
}

// Part k of a tile in the workspace.
__device__ __forceinline__ const float *part_of_tile(const RunStart &run, const TileWork &t, const float *parts, uint32_t c0, uint32_t k, uint32_t floats) {
  return parts + (size_t)slot_of_part(run, t, c0, k) * floats;
}

}  // namespace
