// The rows of a layer's q|k|v projection on their way into attention, one pass: RMSNorm of every query and key head, position
// rotation, queries out in the cache's type, keys and values into the pages of the sequences they belong to.
//
//   y = x / sqrt(mean(x^2) + eps) * w;   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * frequency_j
//
// A thread holds the two vectors that rotate into one another (halves: values j.. and j + rope_dims / 2..; neighbours: 2 V consecutive
// values) and a group of lanes one head, so a head is read once and its mean of squares is a few shuffles.  A CTA takes a row or a few of
// them; cosines and sines are made once per row for all of its heads, from the angle in half turns reduced in 64 bits: positions of
// millions lose nothing, and the reduced angle goes to sincospif in 32.  Sums and rotations in fp32, one rounding at the end.
#include <cuda_runtime.h>

#include "attention.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace {

constexpr uint32_t KV_THREADS = 256;
constexpr uint32_t KV_ROWS = 4;  // rows of a CTA at most

// V values as they lie in memory.
template <typename T, int V>
struct Raw {
  static constexpr int BYTES = sizeof(T) * V;
  __align__(16) T t[V];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; i++) reinterpret_cast<uint4 *>(t)[i] = *(reinterpret_cast<const uint4 *>(p) + i);
    } else if constexpr (BYTES == 8) {
      reinterpret_cast<uint2 *>(t)[0] = *reinterpret_cast<const uint2 *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) t[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = Num<T>::f(t[i]);
  }
};
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *p, float (&x)[V]) {
  Raw<T, V> r;
  r.load(p);
  r.get(x);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[V]) {
  __align__(16) T t[V];
#pragma unroll
  for (int i = 0; i < V; i++) t[i] = Num<T>::one(x[i]);
  if constexpr (sizeof(T) * V == 16)
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(t);
  else if constexpr (sizeof(T) * V == 8)
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(t);
  else {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = t[i];
  }
}

struct KvParams {
  AttnLayer a;
  KvBatchDev kv;
  QkvRowsDev r;
  uint32_t *status;
  uint32_t rows;        // of a CTA
  uint32_t head_step;   // heads of a CTA
  uint32_t group;       // lanes of a head, a power of two
};

// IN: the rows' type, OUT: the cache's and q_out's, V: values of a vector.
template <typename IN, typename OUT, int V>
__global__ void __launch_bounds__(KV_THREADS) k_kv_append(const KvParams p) {
  extern __shared__ float2 s_turn[];  // [rows][rope_dims / 2] cosine and sine
  __shared__ uint64_t s_place[KV_ROWS];  // the row's token in the pages, in values
  __shared__ int32_t s_pos[KV_ROWS];     // and its position; -1: no place
  const AttnLayer &a = p.a;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row0 = blockIdx.x * p.rows, n_rows = min(p.rows, p.kv.n_rows - row0);
  const uint32_t heads = a.q_heads + 2 * a.kv_heads, h0 = blockIdx.y * p.head_step, h1 = min(heads, h0 + p.head_step);
  // The thread's part of the unit'th (row, head) of the CTA: pair m of the head's vectors.  Behind the rotated values neighbours pair up, of which
  // the last may have no second.
  const uint32_t sub = tid & (p.group - 1), unit0 = tid / p.group, units = KV_THREADS / p.group;
  const uint32_t n_heads = h1 - h0, D = a.head_dim, half = a.rope_dims / 2;
  constexpr int STEPS = V == 1 ? 4 : 1;  // V == 1: 32 lanes take up to 4 pairs each
  uint32_t at[STEPS][2];
#pragma unroll
  for (int k = 0; k < STEPS; k++) {
    const uint32_t m = sub + k * p.group, rot = a.rope_dims / (2 * V);
    at[k][0] = m < rot && !a.rope_pairs ? m * V : 2 * m * V;
    at[k][1] = at[k][0] + (m < rot && !a.rope_pairs ? half : V);
  }
  Raw<IN, V> next[STEPS][2];
  auto ask = [&](uint32_t u) {
    if (u >= n_rows * n_heads) return;
    const uint32_t r = n_rows == 1 ? 0 : u / n_heads, h = h0 + u - r * n_heads;
    const uint64_t row = row0 + r;
    const IN *src = h < a.q_heads ? (const IN *)p.r.q + row * p.r.q_stride + (uint64_t)h * D
                    : h < a.q_heads + a.kv_heads ? (const IN *)p.r.k + row * p.r.k_stride + (uint64_t)(h - a.q_heads) * D
                                                 : (const IN *)p.r.v + row * p.r.v_stride + (uint64_t)(h - a.q_heads - a.kv_heads) * D;
    if (h < a.q_heads && !p.r.q) return;
#pragma unroll
    for (int k = 0; k < STEPS; k++)
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (at[k][e] < D) next[k][e].load(src + at[k][e]);
  };
  grid_dep_wait();
  grid_dep_launch();
  ask(unit0);  // while positions and places are looked up
  if (warp < n_rows) {  // a warp finds a row's sequence: the last one that starts at the row or before it
    const uint32_t row = row0 + warp;
    uint32_t starts = 0;
    for (uint32_t s = lane; s < p.kv.n_seqs; s += 32) starts += __ldg(p.kv.row_start + s) <= row;
    const uint32_t seq = __reduce_add_sync(0xFFFFFFFFu, starts);
    int32_t pos = -1;
    uint64_t place = 0;
    if (lane == 0 && seq > 0) {
      uint32_t first, n, len;
      seq_rows(p.kv, seq - 1, &first, &n, &len);
      const uint32_t behind = first + n - row;  // this row and those after it: 1 for the newest
      if (row < first + n && behind <= len) {
        const uint32_t at = len - behind, slot = at / a.page_tokens;
        uint32_t page = 0xFFFFFFFFu;
        if (slot < p.kv.table_stride) page = __ldg(p.kv.page_table + (uint64_t)(seq - 1) * p.kv.table_stride + slot);
        if (page < p.kv.n_pages) {
          pos = (int32_t)at;
          place = page * p.kv.page_stride + (uint64_t)(at - slot * a.page_tokens) * p.kv.token_stride;
        }
      }
      if (row < first + n && pos < 0) atomicOr(p.status, MER_DEVSTAT_BAD_CACHE);
    }
    if (lane == 0) s_pos[warp] = pos, s_place[warp] = place;
  }
  __syncthreads();
  for (uint32_t i = tid; i < n_rows * half; i += KV_THREADS) {
    const uint32_t r = i / half, j = i - r * half;
    if (s_pos[r] < 0) continue;
    const double turns = (double)s_pos[r] * __ldg(a.turns + j);
    float sin, cos;
    sincospif((float)(turns - 2.0 * rint(0.5 * turns)), &sin, &cos);
    s_turn[i] = make_float2(cos * a.rope_scale, sin * a.rope_scale);
  }
  __syncthreads();

  // every group of lanes makes the same number of steps, so that the shuffles of a warp meet
  for (uint32_t u0 = 0; u0 < n_rows * n_heads; u0 += units) {
    const uint32_t u = u0 + unit0, r = n_rows == 1 ? 0 : u / n_heads, h = h0 + u - r * n_heads;
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
    const bool on = u < n_rows * n_heads && s_pos[r] >= 0 && (!is_q || p.r.q);
    const uint32_t head = is_q ? h : is_k ? h - a.q_heads : h - a.q_heads - a.kv_heads;
    const uint64_t row = row0 + r;
    OUT *dst = nullptr;
    if (on)
      dst = is_q ? (OUT *)p.r.q_out + row * p.r.q_out_stride + (uint64_t)head * D
                 : (OUT *)(is_k ? p.kv.k_pages : p.kv.v_pages) + s_place[r] + head * p.kv.head_stride;
    float x[STEPS][2][V];
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < STEPS; k++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        if (on && at[k][e] < D)
          next[k][e].get(x[k][e]);
        else
#pragma unroll
          for (int i = 0; i < V; i++) x[k][e][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) sq = fmaf(x[k][e][i], x[k][e][i], sq);
      }
    ask(u + units);
    const float *w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    for (uint32_t d = 1; d < p.group; d *= 2) sq += __shfl_xor_sync(0xFFFFFFFFu, sq, d);
    const float unit = w ? rsqrtf(sq / (float)D + a.norm_eps) : 1.0f;
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
      const uint32_t m = sub + k * p.group, rot = a.rope_dims / (2 * V);
      if (on && w) {
#pragma unroll
        for (int e = 0; e < 2; e++)
          if (at[k][e] < D) {
            float g[V];
            load_vec<float, V>(w + at[k][e], g);
#pragma unroll
            for (int i = 0; i < V; i++) x[k][e][i] *= unit * g[i];
          }
      }
      if (on && (is_q || is_k) && m < rot) {
        const float2 *turn = s_turn + r * half;
        if (!a.rope_pairs || V == 1) {
#pragma unroll
          for (int i = 0; i < V; i++) {
            const float2 t = turn[m * V + i];
            const float first = x[k][0][i], second = x[k][1][i];
            x[k][0][i] = first * t.x - second * t.y;
            x[k][1][i] = first * t.y + second * t.x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i + 1 < V; i += 2) {
              const float2 t = turn[(at[k][e] + i) / 2];
              const float first = x[k][e][i], second = x[k][e][i + 1];
              x[k][e][i] = first * t.x - second * t.y;
              x[k][e][i + 1] = first * t.y + second * t.x;
            }
        }
      }
    }
    // q may be rotated in place: all of a head's values are in registers before its first store, and no other thread asks for them
    __syncwarp();
    if (on) {
#pragma unroll
      for (int k = 0; k < STEPS; k++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          if (at[k][e] < D) store_vec<OUT, V>(dst + at[k][e], x[k][e]);
    }
  }
}

// Whether `v` values of `size` bytes from `p`, `stride` apart, can be moved as one vector.
bool vec_ok(const void *p, uint64_t stride, uint32_t v, uint32_t size) {
  const uint32_t bytes = v * size < 16 ? v * size : 16;
  return p == nullptr || ((uintptr_t)p % bytes == 0 && stride * size % bytes == 0);
}

template <typename IN, typename OUT, int V>
cudaError_t launch_kv(KvParams &p, dim3 grid, size_t smem, cudaStream_t s) {
  return launch_overlapped(k_kv_append<IN, OUT, V>, grid, KV_THREADS, smem, s, false, p);
}
template <typename IN, typename OUT>
cudaError_t launch_kv(KvParams &p, uint32_t v, dim3 grid, size_t smem, cudaStream_t s) {
  return v == 8 ? launch_kv<IN, OUT, 8>(p, grid, smem, s) : v == 4 ? launch_kv<IN, OUT, 4>(p, grid, smem, s) : launch_kv<IN, OUT, 1>(p, grid, smem, s);
}
template <typename IN>
cudaError_t launch_kv(KvParams &p, uint32_t v, dim3 grid, size_t smem, cudaStream_t s) {
  return p.a.cache_type == MER_VALUE_F16 ? launch_kv<IN, __half>(p, v, grid, smem, s) : launch_kv<IN, __nv_bfloat16>(p, v, grid, smem, s);
}

}  // namespace

cudaError_t launch_kv_append(const AttnLayer &a, const KvBatchDev &kv, const QkvRowsDev &r, uint32_t *status, int sm_count, cudaStream_t s) {
  KvParams p{a, kv, r, status, 1, 0, 0};
  const uint32_t in = r.type == MER_VALUE_F32 ? 4 : 2, heads = a.q_heads + 2 * a.kv_heads;
  // the widest vector that neither a rotated pair nor an address cuts
  uint32_t v = 8;
  auto fits = [&](uint32_t n) {
    return (a.rope_pairs ? a.rope_dims : a.rope_dims / 2) % n == 0 && a.rope_dims % (2 * n) == 0 && vec_ok(r.q, r.q_stride, n, in) && vec_ok(r.k, r.k_stride, n, in) && vec_ok(r.v, r.v_stride, n, in) &&
           vec_ok(r.q_out, r.q_out_stride, n, 2);
  };
  while (v > 1 && !fits(v)) v = v == 8 ? 4 : 1;
  const uint32_t pairs = (a.head_dim / v + 1) / 2;
  p.group = 1;
  while (p.group < pairs && p.group < 32) p.group *= 2;
  const uint32_t units = KV_THREADS / p.group;
  // A few rows: a CTA takes one pass of one row's heads, so that every load is in flight at once.  Many: several rows, whose cosines and sines are
  // made together.
  p.rows = (uint64_t)kv.n_rows * heads >= (uint64_t)sm_count * 16 * units ? KV_ROWS : 1;
  p.head_step = p.rows == 1 ? (heads + (heads + units - 1) / units - 1) / ((heads + units - 1) / units) : heads;
  const dim3 grid((kv.n_rows + p.rows - 1) / p.rows, (heads + p.head_step - 1) / p.head_step);
  const size_t smem = (size_t)p.rows * (a.rope_dims / 2) * sizeof(float2);
  return r.type == MER_VALUE_F32   ? launch_kv<float>(p, v, grid, smem, s)
         : r.type == MER_VALUE_F16 ? launch_kv<__half>(p, v, grid, smem, s)
                                   : launch_kv<__nv_bfloat16>(p, v, grid, smem, s);
}
