// Attention of few new rows over a paged cache: single tokens, drafts.  Any head size up to 256 in steps of 8.
//
//   o = sum_j 2^(s_j - m) v_j / (sum_j 2^(s_j - m) [+ 2^(sink - m)]),  s_j = q . k_j * scale * log2 e,  m = max_j s_j
//
// in one pass over the keys with the running maximum and sum of every row.  What bounds it is reading the cache: per 16 tokens 16 * 2 *
// head_dim values for at most 32 rows of work.  So a warp is a stream of its own: it copies the next chunks of 16 tokens (rows of the pages,
// 16 bytes a lane, swizzled) into a ring that no other warp sees, multiplies the one that has landed (mma.sync on 16 x 16 tiles; at this rate of
// operations the legacy tensor path is idle most of the time) and keeps maximum, sum and output of its own tokens in registers: no barrier
// in the loop.  The warps' results are joined in shared memory at the end of a tile, those of several CTAs through the workspace (attention.cuh).
// The weights go to the second product in the cache's type, 2^-9 (bf16) or 2^-12 (f16) of each at most, like the values they multiply; sums are fp32.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"
#include "attend_join.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace {

struct AttendParams {
  AttnLayer a;
  KvBatchDev kv;
  const void *q;
  void *out;
  uint64_t q_stride, out_stride;
  AttnWorkspace ws;
  uint32_t max_rows;  // sequences with more rows are another kernel's
};

// Rows of a tile are MT * 16, warps NW, chunks in flight per warp ST.
template <int DP>
struct StreamShape {
  static constexpr int NW = DP == 256 ? 4 : 8, ST = DP == 64 ? 6 : 3;
  static constexpr uint32_t KB = NW * 16, THREADS = NW * 32, CHUNK = 2 * 16 * DP * 2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4_trans(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte piece `c` of row `r`; eight rows of one column of pieces lie in eight different bank groups.
template <int DP>
__device__ __forceinline__ uint32_t piece(uint32_t r, uint32_t c) {
  return r * (DP * 2) + ((c ^ (r & 7)) << 4);
}

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(StreamShape<DP>::THREADS, 1) k_attend_stream(const AttendParams p) {
  using S = StreamShape<DP>;
  constexpr int NW = S::NW, ST = S::ST, R = MT * 16;
  constexpr uint32_t KB = S::KB, THREADS = S::THREADS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_work[THREADS / 32 + 4];
  __shared__ uint32_t s_flag;
  uint8_t *s_q = smem;                               // [R][DP], swizzled
  uint8_t *s_ring = smem + R * DP * 2;               // [NW][ST][k, v][16][DP]
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t D = p.a.head_dim, page_tokens = p.a.page_tokens, window = p.a.window;
  const TileShape ts(p.a.q_heads, p.a.kv_heads, R);
  grid_dep_wait();
  grid_dep_launch();
  const RunStart run = find_run<KB, THREADS>(p.kv, ts, window, 0, p.max_rows, blockIdx.x, gridDim.x, 1, s_work);
  if (blockIdx.x == 0) clear_rows_without_place<T, THREADS>(p.a, p.kv, 0, p.max_rows, (T *)p.out, p.out_stride, p.ws.status);
  if (blockIdx.x >= run.parts) return;
  RunWalk<KB> walk(p.kv, ts, window, 0, p.max_rows, run);
  const float to_log2 = p.a.scale * LOG2E;
  const uint32_t ring = smem_u32(s_ring) + warp * (ST * S::CHUNK), q_addr = smem_u32(s_q);

  TileWork t;
  while (walk.next(&t)) {
    const uint32_t rows = t.tokens * t.heads;
    const uint32_t end = t.past + t.token0 + t.tokens;  // behind the last token that a row of the tile sees
    const uint32_t start = window && t.past + t.token0 + 1 > window ? t.past + t.token0 + 1 - window : 0;
    const uint32_t *pages = p.kv.page_table + (uint64_t)t.seq * p.kv.table_stride;
    // ---- the ring: lanes 0 .. 15 know where the chunk's tokens lie, one chunk ahead
    uint32_t bad = 0;
    auto look_up = [&](uint32_t blk) -> uint64_t {  // the lane's token in the pages, in values; ~0: not to be read
      const uint32_t key = blk * KB + warp * 16 + (lane & 15);
      if (blk >= t.hi || key < start || key >= end) return ~0ull;
      const uint32_t slot = key / page_tokens;
      const uint32_t page = slot < p.kv.table_stride ? __ldg(pages + slot) : 0xFFFFFFFFu;
      if (page >= p.kv.n_pages) {
        bad = 1;
        return ~0ull;
      }
      return page * p.kv.page_stride + (uint64_t)(key - slot * page_tokens) * p.kv.token_stride + t.kv_head * p.kv.head_stride;
    };
    auto issue = [&](uint64_t place, uint32_t stage) {
      const uint32_t dst = ring + stage * S::CHUNK;
#pragma unroll
      for (int i = 0; i < DP / 16; i++) {
        const uint32_t idx = i * 32 + lane, r = idx / (DP / 8), c = idx % (DP / 8);
        const uint64_t at = __shfl_sync(0xFFFFFFFFu, place, r);
        const bool in = at != ~0ull && c * 8 < D;
        const uint64_t off = in ? at + c * 8 : 0;
        cp_async16(dst + piece<DP>(r, c), (const T *)p.kv.k_pages + off, in ? 16 : 0);
        cp_async16(dst + 16 * DP * 2 + piece<DP>(r, c), (const T *)p.kv.v_pages + off, in ? 16 : 0);
      }
    };
    uint64_t ahead = look_up(t.lo);
#pragma unroll
    for (int i = 0; i < ST - 1; i++) {
      const uint64_t place = ahead;
      ahead = look_up(t.lo + i + 1);
      if (t.lo + i < t.hi) issue(place, i);
      cp_async_commit();
    }
    // ---- queries, while the first chunks are on their way
    for (uint32_t i = tid; i < R * (DP / 8); i += THREADS) {
      const uint32_t r = i / (DP / 8), c = i % (DP / 8), tok = r / t.heads, h = r - tok * t.heads;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows && c * 8 < D)
        v = __ldg(reinterpret_cast<const uint4 *>((const T *)p.q + (uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + h) * D + c * 8));
      *reinterpret_cast<uint4 *>(s_q + piece<DP>(r, c)) = v;
    }
    __syncthreads();
    // tokens that the lane's rows see: (first, last] of each
    uint32_t last[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int e = 0; e < 2; e++) last[mt][e] = t.past + t.token0 + min(mt * 16 + e * 8 + lane / 4, rows - 1) / t.heads;
    float o[MT][DP / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
      for (int i = 0; i < DP / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[mt][i][e] = 0.0f;
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.0f;
    }
    uint32_t stage = 0, fill = ST - 1;
    for (uint32_t blk = t.lo; blk < t.hi; blk++) {
      {
        const uint64_t place = ahead;
        ahead = look_up(blk + ST);
        if (blk + ST - 1 < t.hi) issue(place, fill);
        cp_async_commit();
        fill = fill + 1 == ST ? 0 : fill + 1;
      }
      cp_async_wait<ST - 1>();
      __syncwarp();
      const uint32_t key0 = blk * KB + warp * 16, base = ring + stage * S::CHUNK;
      stage = stage + 1 == ST ? 0 : stage + 1;
      if (key0 >= end || key0 + 16 <= start) continue;
      float s[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[mt][n][e] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; kk++) {
        uint32_t kf[4];
        ldm4(kf, base + piece<DP>((lane / 16) * 8 + (lane & 7), kk * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          uint32_t qf[4];
          ldm4(qf, q_addr + piece<DP>(mt * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), kk * 2 + (lane >> 4)));
          mma16816<T>(s[mt][0], qf, kf[0], kf[1]);
          mma16816<T>(s[mt][1], qf, kf[2], kf[3]);
        }
      }
      uint32_t pf[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        float top[2] = {-INFINITY, -INFINITY};
        const uint32_t key = key0 + (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t at = key + n * 8 + (e & 1), see = last[mt][e >> 1];
            const bool seen = at <= see && (window == 0 || at + window > see);
            s[mt][n][e] = seen ? s[mt][n][e] * to_log2 : -INFINITY;
            top[e >> 1] = fmaxf(top[e >> 1], s[mt][n][e]);
          }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xFFFFFFFFu, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xFFFFFFFFu, top[e], 2));
          top[e] = fmaxf(top[e], m[mt][e]);
        }
        const bool moved = top[0] != m[mt][0] || top[1] != m[mt][1];
        float less[2];
#pragma unroll
        for (int e = 0; e < 2; e++) less[e] = top[e] == -INFINITY ? 0.0f : top[e] - P_SHIFT;
        if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float f = m[mt][e] == -INFINITY ? 0.0f : exp2_approx(m[mt][e] - top[e]);
            l[mt][e] *= f;
            m[mt][e] = top[e];
#pragma unroll
            for (int i = 0; i < DP / 8; i++) o[mt][i][2 * e] *= f, o[mt][i][2 * e + 1] *= f;
          }
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            s[mt][n][e] = exp2_approx(s[mt][n][e] - less[e >> 1]);
            l[mt][e >> 1] += s[mt][n][e];
          }
        pf[mt][0] = Num<T>::pack(s[mt][0][0], s[mt][0][1]);
        pf[mt][1] = Num<T>::pack(s[mt][0][2], s[mt][0][3]);
        pf[mt][2] = Num<T>::pack(s[mt][1][0], s[mt][1][1]);
        pf[mt][3] = Num<T>::pack(s[mt][1][2], s[mt][1][3]);
      }
      const uint32_t vbase = base + 16 * DP * 2;
#pragma unroll
      for (int dn = 0; dn < DP / 16; dn++) {
        uint32_t vf[4];
        ldm4_trans(vf, vbase + piece<DP>(((lane >> 3) & 1) * 8 + (lane & 7), dn * 2 + (lane >> 4)));
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          mma16816<T>(o[mt][2 * dn], pf[mt], vf[0], vf[1]);
          mma16816<T>(o[mt][2 * dn + 1], pf[mt], vf[2], vf[3]);
        }
      }
    }
    cp_async_wait<0>();
    if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
    // ---- the warps' results: [warp][row] maximum and sum, [warp][row][DP] output, where the rings were
    float *s_m = reinterpret_cast<float *>(s_ring), *s_l = s_m + NW * R, *s_o = s_l + NW * R;
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float sum = l[mt][e];
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
        const uint32_t r = mt * 16 + e * 8 + lane / 4;
        if ((lane & 3) == 0) s_m[warp * R + r] = m[mt][e], s_l[warp * R + r] = sum;
#pragma unroll
        for (int i = 0; i < DP / 8; i++)
          *reinterpret_cast<float2 *>(s_o + ((size_t)warp * R + r) * DP + i * 8 + (lane & 3) * 2) = make_float2(o[mt][i][2 * e], o[mt][i][2 * e + 1]);
      }
    __syncthreads();
    const bool whole = t.lo == t.tile_lo && t.hi == t.tile_hi;
    float *part = p.ws.parts + (size_t)part_slot(run, t, blockIdx.x) * part_floats(R, DP);
    for (uint32_t i = tid; i < rows * (DP / 4); i += THREADS) {
      const uint32_t r = i / (DP / 4), c = i % (DP / 4) * 4;
      float top = -INFINITY, sum = 0.0f;
      float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < NW; w++) top = fmaxf(top, s_m[w * R + r]);
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float mw = s_m[w * R + r], f = mw == -INFINITY ? 0.0f : exp2_approx(mw - top);
        const float4 v = *reinterpret_cast<const float4 *>(s_o + ((size_t)w * R + r) * DP + c);
        sum = fmaf(f, s_l[w * R + r], sum);
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
      }
      if (whole) {
        store_row<T>(p.a, t, r, c, top, sum, acc, (T *)p.out, p.out_stride);
      } else {
        if (c == 0) part[r] = top, part[R + r] = sum;
        *reinterpret_cast<float4 *>(part + 2 * R + (size_t)r * DP + c) = acc;
      }
    }
    __syncthreads();
    if (!whole) {
      join_parts<T, R, DP, THREADS>(p.a, t, run, rows, p.ws, (T *)p.out, p.out_stride, &s_flag, [] { __syncthreads(); });
      __syncthreads();
    }
  }
}

template <typename T, int DP, int MT>
cudaError_t launch_stream(const AttendParams &p, int sm_count, cudaStream_t s) {
  using S = StreamShape<DP>;
  constexpr size_t SMEM = (size_t)MT * 16 * DP * 2 + (size_t)S::NW * S::ST * S::CHUNK;
  static_assert((size_t)S::NW * MT * 16 * (DP + 2) * 4 <= (size_t)S::NW * S::ST * S::CHUNK, "the warps' results lie in the rings");
  const cudaError_t e = cudaFuncSetAttribute(k_attend_stream<T, DP, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
  if (e != cudaSuccess) return e;
  return launch_overlapped(k_attend_stream<T, DP, MT>, dim3(sm_count), S::THREADS, SMEM, s, false, p);
}
template <typename T>
cudaError_t launch_stream(const AttendParams &p, bool two, int sm_count, cudaStream_t s) {
  if (p.a.head_dim <= 64) return two ? launch_stream<T, 64, 2>(p, sm_count, s) : launch_stream<T, 64, 1>(p, sm_count, s);
  if (p.a.head_dim <= 128) return two ? launch_stream<T, 128, 2>(p, sm_count, s) : launch_stream<T, 128, 1>(p, sm_count, s);
  return launch_stream<T, 256, 1>(p, sm_count, s);
}

}  // namespace

size_t attend_part_floats(int sm_count) {
  return std::max({(size_t)2 * sm_count * part_floats(32, 128), (size_t)2 * sm_count * part_floats(16, 256), attend_tc_part_floats(sm_count)});
}
size_t attend_counts(int sm_count) { return (size_t)sm_count; }

cudaError_t launch_attend(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                          int sm_count, cudaStream_t s, int *launches) {
  // Rows of a sequence's tile on average.  16 and 32 are the tiles of the streaming kernel; beyond those it would read the cache once
  // per 32 rows, and multiply them at the legacy rate.
  const uint64_t rows = (uint64_t)(a.q_heads / a.kv_heads) * ((kv.n_rows + kv.n_seqs - 1) / kv.n_seqs);
  *launches += 1;
  if (rows > 32 && a.head_dim <= 128) return launch_attend_tc(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
  AttendParams p{a, kv, q, out, q_stride, out_stride, ws, 0xFFFFFFFFu};
  return a.cache_type == MER_VALUE_F16 ? launch_stream<__half>(p, rows > 16, sm_count, s) : launch_stream<__nv_bfloat16>(p, rows > 16, sm_count, s);
}
