// The rows of a layer's q|k|v projection on their way into attention, one pass: RMSNorm of every query and key head, position
// rotation, queries out in the cache's type, keys and values into the pages of the sequences they belong to.
//
//   y = x / sqrt(mean(x^2) + eps) * w;   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * frequency_j
//
// A thread holds the two vectors that rotate into one another (halves: values j.. and j + rope_dims / 2..; neighbours: 2 V consecutive
// values) and a group of lanes one head, so a head is read once and its mean of squares is a few shuffles.  A CTA is a warp, which has a row,
// or some of its heads, and goes through them a few at a time: cosines, sines and weights stay in its registers, and the heads to come are on
// their way.  Angles are made in half turns reduced in 64 bits: positions of millions lose nothing, and the reduced angle goes to sincospif in
// 32.  Sums and rotations in fp32, two values an instruction; one rounding at the end.
// What bounds it: memory for thousands of rows, with the instructions close behind (200 a step of 16 values a thread, 300 for a row's place and
// cosines), which bound rows of few heads: 20781 of 2 + 2 heads of 128 28 us, where the bytes take 6.5; queries, keys and values take whole steps each, so that 2, 1 and 1 heads
// are three steps which use half, a quarter and a quarter of the lanes.  A warp to a CTA, because a CTA's place is
// free only when its last warp has ended: 13411 rows of 32 + 2 * 8 heads of 128 in f16 60.3 us with CTAs of one warp, 64.1 of two, 67.8 of four,
// 78.1 of eight (two steps ahead each; three: 57.0, 5.8 TB/s).  With a CTA for four rows, whose threads took any head and read cosines and weights
// again for each, 69.5; with two rows to a warp, whose state takes 122 registers instead of 106, 68.8.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"
#include "kernels.h"
#include "pack2.cuh"
#include "ptx.cuh"

namespace {

constexpr int AHEAD = 3;          // steps whose values a warp has asked for (2: 60.3 us, 4: 61.0, where registers cost warps)

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
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < BYTES / 2; i++) reinterpret_cast<uint16_t *>(t)[i] = 0;
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = Num<T>::f(t[i]);
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[V]) {
  if constexpr (V % 2 == 0) {
    uint32_t t[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) t[i] = Num<T>::pack(x[2 * i], x[2 * i + 1]);
    if constexpr (V == 8)
      *reinterpret_cast<uint4 *>(p) = make_uint4(t[0], t[1], t[2], t[3]);
    else
      *reinterpret_cast<uint2 *>(p) = make_uint2(t[0], t[1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = Num<T>::one(x[i]);
  }
}
// a[i] * b[i], two at a time.
template <int V>
__device__ __forceinline__ void times(float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) unpack2(mul2(pack2(a[i], a[i + 1]), pack2(b[i], b[i + 1])), a[i], a[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) a[i] *= b[i];
  }
}
// (a, b) -> (a c - b s, a s + b c)
template <int V>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const uint64_t a2 = pack2(a[i], a[i + 1]), b2 = pack2(b[i], b[i + 1]), c2 = pack2(c[i], c[i + 1]), s2 = pack2(s[i], s[i + 1]);
      unpack2(fma2(pack2(-b[i], -b[i + 1]), s2, mul2(a2, c2)), a[i], a[i + 1]);
      unpack2(fma2(b2, c2, mul2(a2, s2)), b[i], b[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i], b[i] = x * s[i] + y * c[i];
    }
  }
}

struct KvParams {
  AttnLayer a;
  KvBatchDev kv;
  QkvRowsDev r;
  uint32_t *status;
  uint32_t group;             // lanes of a head, a power of two
  uint32_t q_steps, kv_steps; // steps of 32 / group heads
  uint32_t chunks, each;      // warps of a row, and steps of each
  float per_value;            // 1 / head_dim
};

// IN: the rows' type, OUT: the cache's and q_out's, V: values of a vector.
template <typename IN, typename OUT, int V>
__global__ void __launch_bounds__(32) k_kv_append(const KvParams p) {
  extern __shared__ float2 turns[];  // [rope_dims / 2] cosine and sine
  const AttnLayer &a = p.a;
  const uint32_t lane = threadIdx.x, row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  const uint32_t D = a.head_dim, half = a.rope_dims / 2, sub = lane & (p.group - 1), of = lane / p.group, heads = 32 / p.group;
  // Pair m of a head's vectors.  Behind the rotated values neighbours pair up, of which the last may have no second.
  constexpr int STEPS = V == 1 ? 4 : 1;  // V == 1: 32 lanes take up to 4 pairs each
  const uint32_t rot = a.rope_dims / (2 * V);
  uint32_t at[STEPS][2];
#pragma unroll
  for (int k = 0; k < STEPS; k++) {
    const uint32_t m = sub + k * p.group;
    at[k][0] = m < rot && !a.rope_pairs ? m * V : 2 * m * V;
    at[k][1] = at[k][0] + (m < rot && !a.rope_pairs ? half : V);
  }
  const uint32_t steps = p.q_steps + 2 * p.kv_steps, first_step = chunk * p.each, end_step = min(steps, first_step + p.each);
  // Step i has the heads (i - the part's first step) * heads + of of the queries, keys or values.
  const uint32_t k_first = p.q_steps, v_first = p.q_steps + p.kv_steps;
  auto part_of = [&](uint32_t i) { return i < k_first ? 0u : i < v_first ? 1u : 2u; };
  auto head_of = [&](uint32_t i, uint32_t part) { return (i - (part == 0 ? 0 : part == 1 ? k_first : v_first)) * heads + of; };
  const IN *const q_src = (const IN *)p.r.q + row * p.r.q_stride, *const k_src = (const IN *)p.r.k + row * p.r.k_stride, *const v_src = (const IN *)p.r.v + row * p.r.v_stride;
  Raw<IN, V> ahead[AHEAD][STEPS][2];
#pragma unroll
  for (int i = 0; i < AHEAD * STEPS * 2; i++) (&ahead[0][0][0])[i].clear();  // what is never asked for stays zero
  auto is_there = [&](uint32_t part, uint32_t head) { return part == 0 ? head < a.q_heads && p.r.q : head < a.kv_heads; };
  auto ask = [&](uint32_t i, Raw<IN, V>(&next)[STEPS][2]) {
    if (i >= end_step) return;
    const uint32_t part = part_of(i), head = head_of(i, part);
    if (!is_there(part, head)) return;
    const IN *src = (part == 0 ? q_src : part == 1 ? k_src : v_src) + head * D;
#pragma unroll
    for (int k = 0; k < STEPS; k++)
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (at[k][e] < D) next[k][e].load(src + at[k][e]);
  };
  grid_dep_wait();
  grid_dep_launch();
#pragma unroll
  for (int d = 0; d < AHEAD; d++) ask(first_step + d, ahead[d]);  // while position and place are looked up
  // The row's sequence is the last one that starts at the row or before it: the lanes read all starts and lengths in one round trip.
  uint32_t pos = 0xFFFFFFFFu;
  uint64_t place = 0;
  {
    uint32_t s0 = 0, s1 = p.kv.n_seqs;
    while (s1 - s0 > 128) {  // many: the lanes look at 32 starts at a time
      const uint32_t step = (s1 - s0 + 31) / 32, s = s0 + lane * step;
      const uint32_t before = __popc(__ballot_sync(0xFFFFFFFFu, s < s1 && p.kv.row_start[s] <= row));
      if (before == 0) return;
      s0 += (before - 1) * step, s1 = min(s1, s0 + step);
    }
    uint32_t seq = 0, end = 0, len = 0;  // seq: its number + 1
    for (uint32_t s = s0 + lane; s < s1; s += 32) {
      const uint32_t start = p.kv.row_start[s], e = p.kv.row_start[s + 1], n = p.kv.kv_len[s];
      if (start <= row) seq = s + 1, end = e, len = n <= p.kv.capacity ? n : 0;
    }
    const uint32_t last = __reduce_max_sync(0xFFFFFFFFu, seq);
    if (last == 0) return;
    const uint32_t from = __ffs(__ballot_sync(0xFFFFFFFFu, seq == last)) - 1;
    end = min(__shfl_sync(0xFFFFFFFFu, end, from), p.kv.n_rows), len = __shfl_sync(0xFFFFFFFFu, len, from);
    if (row >= end) return;  // behind the last sequence
    const uint32_t behind = end - row;  // this row and those after it: 1 for the newest
    if (behind <= len) {
      const uint32_t slot = divided(len - behind, p.kv.page_tokens);
      const uint32_t page = slot < p.kv.table_stride ? p.kv.page_table[(uint64_t)(last - 1) * p.kv.table_stride + slot] : 0xFFFFFFFFu;
      if (page < p.kv.n_pages) {
        pos = len - behind;
        place = page * p.kv.page_stride + (uint64_t)(pos - slot * a.page_tokens) * p.kv.token_stride;
      }
    }
    if (pos == 0xFFFFFFFFu) {
      if (lane == 0) atomicOr(p.status, MER_DEVSTAT_BAD_CACHE);
      return;
    }
  }
  for (uint32_t j = lane; j < half; j += 32) {
    const double x = (double)pos * __ldg(a.turns + j);
    float sin, cos;
    sincospif((float)(x - 2.0 * rint(0.5 * x)), &sin, &cos);
    turns[j] = make_float2(cos * a.rope_scale, sin * a.rope_scale);
  }
  __syncwarp();
  // A thread's cosines and sines: of the pairs across its two vectors, or within each of them.
  constexpr int PAIRS = V == 1 ? 1 : V;
  float c[STEPS][PAIRS], s[STEPS][PAIRS];
#pragma unroll
  for (int k = 0; k < STEPS; k++) {
    const uint32_t m = sub + k * p.group;
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
      // halves: pair m V + i; neighbours: the V pairs of 2 V values; one value a vector: pair m
      const float2 t = m < rot ? turns[m * V + i] : make_float2(1.0f, 0.0f);
      c[k][i] = t.x, s[k][i] = t.y;
    }
  }
  OUT *const q_dst = (OUT *)p.r.q_out + row * p.r.q_out_stride, *const k_dst = (OUT *)p.kv.k_pages + place, *const v_dst = (OUT *)p.kv.v_pages + place;
  float w[STEPS][2][V] = {};
  uint32_t w_part = 3;  // the part whose weights these are
  auto process = [&](uint32_t i, Raw<IN, V>(&next)[STEPS][2]) {
    const uint32_t part = part_of(i), head = head_of(i, part);
    float x[STEPS][2][V];  // of a head that is not there, whatever
#pragma unroll
    for (int k = 0; k < STEPS; k++)
#pragma unroll
      for (int e = 0; e < 2; e++) next[k][e].get(x[k][e]);
    ask(i + AHEAD, next);
    const float *weights = part == 0 ? a.q_norm : part == 1 ? a.k_norm : nullptr;
    if (weights) {
      if (w_part != part) {
        w_part = part;
#pragma unroll
        for (int k = 0; k < STEPS; k++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (at[k][e] < D) {
              Raw<float, V> t;
              t.load(weights + at[k][e]);
              t.get(w[k][e]);
            }
      }
      float sq = 0.0f;
      if constexpr (V % 2 == 0) {
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int v = 0; v < V; v += 2) {
            const uint64_t t = pack2(x[0][e][v], x[0][e][v + 1]);
            sum[e] = fma2(t, t, sum[e]);
          }
        float lo, hi;
        unpack2(add2(sum[0], sum[1]), lo, hi);
        sq = lo + hi;
      } else {
#pragma unroll
        for (int k = 0; k < STEPS; k++) sq += x[k][0][0] * x[k][0][0] + x[k][1][0] * x[k][1][0];
      }
#pragma unroll
      for (uint32_t d = 1; d < 32; d *= 2) {
        const float other = __shfl_xor_sync(0xFFFFFFFFu, sq, d);
        sq += d < p.group ? other : 0.0f;
      }
      const float unit = rsqrtf(fmaf(sq, p.per_value, a.norm_eps));
#pragma unroll
      for (int k = 0; k < STEPS; k++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float u[V];
#pragma unroll
          for (int v = 0; v < V; v++) u[v] = unit;
          times<V>(x[k][e], u);
          times<V>(x[k][e], w[k][e]);
        }
    }
    if (part != 2 && half > 0) {
#pragma unroll
      for (int k = 0; k < STEPS; k++) {
        if (sub + k * p.group >= rot) continue;
        if (V > 1 && a.rope_pairs) {
          // values 2 i and 2 i + 1 of the 2 V are pair i
          float e0[V], e1[V];
#pragma unroll
          for (int v = 0; v < V; v++) e0[v] = x[k][2 * v / V][2 * v % V], e1[v] = x[k][(2 * v + 1) / V][(2 * v + 1) % V];
          turn<V>(e0, e1, c[k], s[k]);
#pragma unroll
          for (int v = 0; v < V; v++) x[k][2 * v / V][2 * v % V] = e0[v], x[k][(2 * v + 1) / V][(2 * v + 1) % V] = e1[v];
        } else {
          turn<V>(x[k][0], x[k][1], c[k], s[k]);
        }
      }
    }
    // q may be rotated in place: all of a head's values are in registers before its first store, and no other thread asks for them
    __syncwarp();
    if (is_there(part, head)) {
      OUT *dst = part == 0 ? q_dst + head * D : (part == 1 ? k_dst : v_dst) + head * p.kv.head_stride;
#pragma unroll
      for (int k = 0; k < STEPS; k++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          if (at[k][e] < D) store_vec<OUT, V>(dst + at[k][e], x[k][e]);
    }
  };
  for (uint32_t i = first_step; i < end_step; i += AHEAD) {
#pragma unroll
    for (int d = 0; d < AHEAD; d++)
      if (i + d < end_step) process(i + d, ahead[d]);
  }
}

// Whether `v` values of `size` bytes from `p`, `stride` apart, can be moved as one vector.
bool vec_ok(const void *p, uint64_t stride, uint32_t v, uint32_t size) {
  const uint32_t bytes = v * size < 16 ? v * size : 16;
  return p == nullptr || ((uintptr_t)p % bytes == 0 && stride * size % bytes == 0);
}

template <typename IN, typename OUT, int V>
cudaError_t launch_kv(KvParams &p, dim3 grid, size_t smem, cudaStream_t s) {
  return launch_overlapped(k_kv_append<IN, OUT, V>, grid, 32, smem, s, false, p);
}
template <typename IN, typename OUT>
cudaError_t launch_kv(KvParams &p, uint32_t v, dim3 grid, size_t smem, cudaStream_t s) {
  if constexpr (sizeof(IN) == 2)
    if (v == 8) return launch_kv<IN, OUT, 8>(p, grid, smem, s);
  return v == 4 ? launch_kv<IN, OUT, 4>(p, grid, smem, s) : launch_kv<IN, OUT, 1>(p, grid, smem, s);
}
template <typename IN>
cudaError_t launch_kv(KvParams &p, uint32_t v, dim3 grid, size_t smem, cudaStream_t s) {
  return p.a.cache_type == MER_VALUE_F16 ? launch_kv<IN, __half>(p, v, grid, smem, s) : launch_kv<IN, __nv_bfloat16>(p, v, grid, smem, s);
}

}  // namespace

cudaError_t launch_kv_append(const AttnLayer &a, const KvBatchDev &kv, const QkvRowsDev &r, uint32_t *status, int sm_count, cudaStream_t s) {
  KvParams p{a, kv, r, status, 1, 0, 0, 1, 0, 1.0f / (float)a.head_dim};
  const uint32_t in = r.type == MER_VALUE_F32 ? 4 : 2;
  // The widest vector up to 16 bytes that neither a rotated pair nor an address cuts.  (Eight fp32 values a vector: 24652 rows of 8 + 2 heads of 128 61 us,
  // 50 so, with 72 registers instead of 121; four f16 values: 13411 rows of 32 + 2 * 8 heads 83 us, 57 with eight.)
  uint32_t v = in == 4 ? 4 : 8;
  auto fits = [&](uint32_t n) {
    return a.rope_dims % (2 * n) == 0 && vec_ok(r.q, r.q_stride, n, in) && vec_ok(r.k, r.k_stride, n, in) && vec_ok(r.v, r.v_stride, n, in) &&
           vec_ok(r.q_out, r.q_out_stride, n, 2);
  };
  while (v > 1 && !fits(v)) v = v == 8 ? 4 : 1;
  const uint32_t pairs = (a.head_dim / v + 1) / 2;
  while (p.group < pairs && p.group < 32) p.group *= 2;
  const uint32_t heads = 32 / p.group;
  p.q_steps = (a.q_heads + heads - 1) / heads, p.kv_steps = (a.kv_heads + heads - 1) / heads;
  // A warp a row, and more of them while there are fewer than 16 an SM: fewer steps one after the other.
  const uint32_t steps = p.q_steps + 2 * p.kv_steps;
  p.chunks = (uint32_t)std::min<uint64_t>(steps, std::max<uint64_t>(1, (uint64_t)sm_count * 16 / kv.n_rows));
  p.each = (steps + p.chunks - 1) / p.chunks;
  p.chunks = (steps + p.each - 1) / p.each;
  const dim3 grid(kv.n_rows * p.chunks);  // one row's warps only where rows are few: below 2^31
  const size_t smem = (size_t)(a.rope_dims / 2) * sizeof(float2);
  return r.type == MER_VALUE_F32   ? launch_kv<float>(p, v, grid, smem, s)
         : r.type == MER_VALUE_F16 ? launch_kv<__half>(p, v, grid, smem, s)
                                   : launch_kv<__nv_bfloat16>(p, v, grid, smem, s);
}
