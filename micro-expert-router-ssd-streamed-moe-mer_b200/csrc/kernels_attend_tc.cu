// Attention of many new rows over a paged cache: prompts, chunks of prompts, steps that mix them with single tokens.  Heads of up to 128 values.
//
// The same one pass as kernels_attend.cu, on tcgen05: a tile is two groups of 128 rows (tokens x heads of a key head), a block 128 tokens.
//
//   S[128 x 128] = Q[128 x d] K[128 x d]^T      both from shared memory, S in tensor memory
//   P = 2^(S * scale - m + shift)               a thread owns a row: its maximum and sum need no other thread
//   O[128 x d] += P[128 x 128] V[128 x d]       P from tensor memory, where it takes the place of S; V's rows run along N
//
//   * Warps 0..3 and 4..7 are the softmax of one group of rows each, warp 8 issues the MMAs, warps 9 and 10 copy.  While one group's
//     softmax runs the tensor core multiplies for the other: [P V of block j, Q K of block j + 1] of one, then of the other.
//   * The reference maximum of a row follows its maximum only when that has grown by more than 2^LAG; then alone the output in tensor memory is rescaled, by
//     the softmax warps themselves.  Until then weights are larger than 1 by up to that factor, which f16 and fp32 hold.  What makes that safe without a
//     barrier: the MMAs complete in order, so the S of block j being there says that the P V of block j - 1 has been added.
//   * Keys and values come as rows of the pages, 16 bytes a lane (cp.async), whatever the page size is, and are written in the
//     swizzle that the MMA reads; a copying warp makes its rows visible to the tensor core (proxy fence) and arrives.
//   * Rows of P that see nothing of a block hold zeros, and what no row sees is filled with zeros instead of being read.
// What bounds it: exponentials and MMAs, 2048 cycles each for a block of both groups at 16 and 8192 a cycle.
// Every wait is bounded; on expiry the CTA latches MER_DEVSTAT_TIMEOUT, stops issuing work, waits (bounded) for what is in flight,
// frees its tensor memory and returns.
#include <cuda_runtime.h>

#include "attend_join.cuh"
#include "attention.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "tmem.cuh"

namespace {

struct TcParams {
  AttnLayer a;
  KvBatchDev kv;
  const void *q;
  void *out;
  uint64_t q_stride, out_stride;
  AttnWorkspace ws;
  uint32_t min_blocks;
};

constexpr uint32_t TC_R = 256, TC_KB = 128, TC_WARPS = 11, TC_THREADS = TC_WARPS * 32, SOFT_THREADS = 256;
constexpr uint32_t TC_MMA = 8, TC_LOAD = 9, TC_LOADERS = 2;
constexpr float LAG = 3.0f;  // with P_SHIFT the largest weight is 2^15
constexpr uint32_t TC_CONTROL = 1024;  // barriers and words in front of the operands

template <int DP>
struct TcShape {
  static constexpr uint32_t SUBS = DP / 64;                // pieces of 64 values of a row
  static constexpr uint32_t STAGE = SUBS * TC_KB * 128;    // keys or values of a block
  static constexpr uint32_t STAGES = DP == 128 ? 5 : 10;
  static constexpr uint32_t QTILE = SUBS * 128 * 128;
  static constexpr size_t SMEM = TC_CONTROL + 1024 + 2 * QTILE + STAGES * STAGE;  // 1024: the operands lie on whole atoms
};

struct TcControl {
  uint64_t full[10], empty[10];  // stages of the ring
  uint64_t q_full, q_empty, s_full[2], p_ready[2], o_full[2], soft, drain;
  uint64_t work[TC_THREADS / 32 + 4];
  uint32_t tmem, flag;
  volatile uint32_t abort;
};
static_assert(sizeof(TcControl) <= TC_CONTROL, "control block");

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void copies_left() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <typename T, int DP>
__global__ void __launch_bounds__(TC_THREADS, 1) k_attend_tc(const TcParams p) {
  using S = TcShape<DP>;
  extern __shared__ __align__(16) uint8_t smem[];
  TcControl &ctl = *reinterpret_cast<TcControl *>(smem);
  const uint32_t operands = (smem_u32(smem) + TC_CONTROL + 1023u) & ~1023u;
  const uint32_t s_q = operands, s_ring = operands + 2 * S::QTILE;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t D = p.a.head_dim, window = p.a.window;
  const TileShape ts(p.a.q_heads, p.a.kv_heads, TC_R);
  if (tid == 0) {
    for (uint32_t i = 0; i < S::STAGES; i++) mbar_init(&ctl.full[i], TC_LOADERS), mbar_init(&ctl.empty[i], 1);
    mbar_init(&ctl.q_full, TC_LOADERS), mbar_init(&ctl.q_empty, 1);
    for (int x = 0; x < 2; x++) mbar_init(&ctl.s_full[x], 1), mbar_init(&ctl.p_ready[x], 4), mbar_init(&ctl.o_full[x], 1);
    mbar_init(&ctl.soft, SOFT_THREADS / 32), mbar_init(&ctl.drain, 1);
    ctl.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  grid_dep_wait();
  grid_dep_launch();
  const RunStart run = find_run<TC_KB, TC_THREADS>(p.kv, ts, window, 0, 0xFFFFFFFFu, blockIdx.x, gridDim.x, p.min_blocks, ctl.work);
  if (blockIdx.x == 0) clear_rows_without_place<T, TC_THREADS>(p.a, p.kv, 0, 0xFFFFFFFFu, (T *)p.out, p.out_stride, p.ws.status);
  if (blockIdx.x >= run.parts) return;
  if (warp == TC_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tm = ctl.tmem;
  // columns: S (and P) of the two groups at 0 and 128, their O at 256 and 256 + DP
  RunWalk<TC_KB> walk(p.kv, ts, window, 0, 0xFFFFFFFFu, run);
  TileWork t;
  // For whole warps, which stay together whatever comes of it.
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    const bool ok = mbar_wait(bar, parity, &ctl.abort);
    if (!ok && !ctl.abort) {
      ctl.abort = 1;
      atomicOr(p.ws.status, MER_DEVSTAT_TIMEOUT);
    }
    return __all_sync(0xFFFFFFFFu, ok) != 0;
  };
  auto aborted = [&] { return __any_sync(0xFFFFFFFFu, ctl.abort) != 0; };

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax: a thread has row x * 128 + (tid & 127) of the tile
    const uint32_t x = warp >> 2, row = tid;
    const uint32_t tm_lane = tm + ((warp & 3) << 21), s_at = tm_lane + x * 128, o_at = tm_lane + 256 + x * DP;
    const float to_log2 = p.a.scale * LOG2E;
    uint32_t blocks = 0, tiles = 0, syncs = 0;  // phases of s_full, o_full, soft
    auto sync = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.soft);
      wait(&ctl.soft, syncs++ & 1);
    };
    while (!aborted() && walk.next(&t)) {
      const uint32_t rows = t.tokens * t.heads;
      const bool active = rows > x * 128;
      const uint32_t first = t.past + t.token0, see = first + min(row, rows - 1) / t.heads;
      const uint32_t least = window && see + 1 > window ? see + 1 - window : 0;  // the row sees least .. see
      float m = -INFINITY, l = 0.0f;
      if (active) {
        // blocks that every row of the group sees whole need no mask
        const uint32_t see0 = first + x * 128 / t.heads, see1 = first + min(x * 128 + 127, rows - 1) / t.heads;
        const uint32_t least1 = window && see1 + 1 > window ? see1 + 1 - window : 0;
        for (uint32_t blk = t.lo; blk < t.hi; blk++, blocks++) {
          if (!wait(&ctl.s_full[x], blocks & 1)) break;
          tm_fence_after();
          float s[128];
          tm_load(s_at, s);
          const uint32_t key0 = blk * TC_KB;
          if (key0 + TC_KB - 1 > see0 || key0 < least1) {
#pragma unroll
            for (int i = 0; i < 128; i++) s[i] = key0 + i <= see && key0 + i >= least ? s[i] : -INFINITY;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 128; i += 4)
#pragma unroll
            for (int e = 0; e < 4; e++) top[e] = fmaxf(top[e], s[i + e]);
          const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * to_log2;
          const bool grow = now > m + LAG || (m == -INFINITY && now > m);
          if (__any_sync(0xFFFFFFFFu, grow)) {
            const float f = grow ? (m == -INFINITY ? 0.0f : exp2_approx(m - now)) : 1.0f;
            if (grow) m = now;
            l *= f;
            if (blk != t.lo) {
              float o[32];
#pragma unroll 1
              for (int c = 0; c < DP; c += 32) {
                tm_load(o_at + c, o);
                uint32_t v[32];
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = __float_as_uint(o[i] * f);
                tm_store(o_at + c, v);
              }
            }
          }
          const float less = m == -INFINITY ? 0.0f : m - P_SHIFT;
          float sum[4] = {0, 0, 0, 0};
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
              const float a = exp2_approx(fmaf(s[h * 64 + 2 * i], to_log2, -less)), b = exp2_approx(fmaf(s[h * 64 + 2 * i + 1], to_log2, -less));
              sum[i & 3] += a + b;
              v[i] = Num<T>::pack(a, b);
            }
            tm_store(s_at + h * 32, v);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tm_wait_store();
          tm_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.p_ready[x]);
        }
      }
      const bool whole = t.lo == t.tile_lo && t.hi == t.tile_hi;
      float *part = p.ws.parts + (size_t)part_slot(run, t, blockIdx.x) * part_floats(TC_R, DP);
      if (active) {
        if (!wait(&ctl.o_full[x], tiles++ & 1)) break;
        tm_fence_after();
        const uint32_t tok = row / t.heads, head = t.head0 + row - tok * t.heads;
        float f = 1.0f;
        if (whole && row < rows) {
          const float total = p.a.sinks ? l + exp2_approx(__ldg(p.a.sinks + head) * LOG2E - m + P_SHIFT) : l;
          f = total == 0.0f ? 0.0f : 1.0f / total;
        }
        T *out = (T *)p.out + (uint64_t)(t.row0 + t.token0 + tok) * p.out_stride + (uint64_t)head * D;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          float o[32];
          __syncwarp();
          tm_load(o_at + c, o);
          if (row >= rows) continue;
          if (whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              const uint4 v = make_uint4(Num<T>::pack(o[i] * f, o[i + 1] * f), Num<T>::pack(o[i + 2] * f, o[i + 3] * f), Num<T>::pack(o[i + 4] * f, o[i + 5] * f),
                                         Num<T>::pack(o[i + 6] * f, o[i + 7] * f));
              if (c + i < (int)D) *reinterpret_cast<uint4 *>(out + c + i) = v;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(part + 2 * TC_R + (size_t)row * DP + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (!whole && row < rows) part[row] = m, part[TC_R + row] = l;
        tm_fence_before();
      }
      if (!whole && !aborted()) join_parts<T, TC_R, DP, SOFT_THREADS>(p.a, t, run, rows, p.ws, (T *)p.out, p.out_stride, &ctl.flag, sync);
    }
  } else if (warp == TC_MMA) {
    // ---------------------------------------------------------------- MMA issue
    const uint32_t leader = tm_elect();
    constexpr uint32_t TYPE = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t BASE = (1u << 4) | (TYPE << 7) | (TYPE << 10) | ((128u >> 4) << 24);
    constexpr uint32_t QK = BASE | ((TC_KB >> 3) << 17), PV = BASE | (1u << 16) | ((DP >> 3) << 17);
    uint32_t stage = 0, phase = 0, tiles = 0, blocks = 0;  // blocks: phases of p_ready[0]; of p_ready[1] the same while its group is active
    uint32_t blocks1 = 0;
    auto next_stage = [&] { stage = stage + 1 == S::STAGES ? 0 : stage + 1, phase ^= stage == 0; };
    auto qk = [&](uint32_t x, uint32_t st) {
#pragma unroll
      for (int k = 0; k < DP / 16; k++)
        tm_mma_ss(leader, tm + x * 128, tm_desc(s_q + x * S::QTILE + (k / 4) * 16384 + (k & 3) * 32, 16),
                  tm_desc(s_ring + st * S::STAGE + (k / 4) * (TC_KB * 128) + (k & 3) * 32, 16), QK, k != 0);
      tm_commit(leader, &ctl.s_full[x]);
    };
    while (!aborted() && walk.next(&t)) {
      const uint32_t groups = t.tokens * t.heads > 128 ? 2 : 1;
      if (!wait(&ctl.q_full, tiles & 1)) break;
      if (!wait(&ctl.full[stage], phase)) break;
      tm_fence_after();
      for (uint32_t x = 0; x < groups; x++) qk(x, stage);
      tm_commit(leader, &ctl.empty[stage]);
      next_stage();
      if (t.lo + 1 == t.hi) tm_commit(leader, &ctl.q_empty);
      bool ok = true;
      for (uint32_t blk = t.lo; blk < t.hi && ok; blk++) {
        const uint32_t v_stage = stage, v_phase = phase;
        const bool more = blk + 1 < t.hi;
        next_stage();
        if (!(ok = wait(&ctl.full[v_stage], v_phase))) break;
        if (more && !(ok = wait(&ctl.full[stage], phase))) break;
        for (uint32_t x = 0; x < groups; x++) {
          if (!(ok = wait(&ctl.p_ready[x], (x ? blocks1 : blocks) & 1))) break;
          tm_fence_after();
#pragma unroll
          for (int k = 0; k < (int)TC_KB / 16; k++)
            tm_mma_ts(leader, tm + 256 + x * DP, tm + x * 128 + k * 8, tm_desc(s_ring + v_stage * S::STAGE + k * 2048, TC_KB * 128), PV, k != 0 || blk != t.lo);
          if (more)
            qk(x, stage);
          else
            tm_commit(leader, &ctl.o_full[x]);
        }
        if (!ok) break;
        blocks++;
        if (groups == 2) blocks1++;
        tm_commit(leader, &ctl.empty[v_stage]);
        if (more) {
          tm_commit(leader, &ctl.empty[stage]);
          next_stage();
          if (blk + 2 == t.hi) tm_commit(leader, &ctl.q_empty);
        }
      }
      if (!ok) break;
      tiles++;
    }
    if (aborted()) {
      tm_commit(leader, &ctl.drain);
      mbar_drain(&ctl.drain, 0, 1000000000ull);
    }
  } else {
    // ---------------------------------------------------------------- copies: warp w has the rows w * 64 .. of a block, and half of the queries
    const uint32_t w = warp - TC_LOAD;
    uint32_t stage = 0, phase = 0, tiles = 0, bad = 0;
    uint64_t *pending[3] = {nullptr, nullptr, nullptr};  // barriers of the copies in flight, the newest first
    auto landed = [&](uint64_t *bar) {
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto settle = [&] {  // everything in flight has landed
      copies_left<0>();
#pragma unroll
      for (int i = 2; i >= 0; i--) {
        if (pending[i]) landed(pending[i]);
        pending[i] = nullptr;
      }
    };
    auto submit = [&](uint64_t *bar) {
      asm volatile("cp.async.commit_group;" ::: "memory");
      copies_left<3>();
      if (pending[2]) landed(pending[2]);
      pending[2] = pending[1], pending[1] = pending[0], pending[0] = bar;
    };
    auto claim = [&](uint64_t *bar, uint32_t parity) {  // nothing is held back while this warp waits
      if (__all_sync(0xFFFFFFFFu, mbar_test(bar, parity))) return true;
      settle();
      return wait(bar, parity);
    };
    constexpr uint32_t PIECES = DP / 8;  // of a row
    while (!aborted() && walk.next(&t)) {
      const uint32_t rows = t.tokens * t.heads;
      if (!claim(&ctl.q_empty, (tiles & 1) ^ 1)) break;
      for (uint32_t i = lane; i < 128 * PIECES; i += 32) {
        const uint32_t r = w * 128 + i / PIECES, c = i % PIECES, tok = r / t.heads, h = r - tok * t.heads;
        const bool in = r < rows && c * 8 < D;
        const T *src = (const T *)p.q;
        if (in) src += (uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + h) * D + c * 8;
        copy16(s_q + w * S::QTILE + (c / 8) * 16384 + (i / PIECES) * 128 + (((c ^ r) & 7) << 4), src, in ? 16 : 0);
      }
      submit(&ctl.q_full);
      tiles++;
      const uint32_t end = t.past + t.token0 + t.tokens;
      const uint32_t start = window && t.past + t.token0 + 1 > window ? t.past + t.token0 + 1 - window : 0;
      const uint32_t *pages = p.kv.page_table + (uint64_t)t.seq * p.kv.table_stride;
      // a lane knows where the tokens w * 64 + lane and + 32 of the block lie, a block ahead
      auto look_up = [&](uint32_t blk, uint32_t half) -> uint64_t {
        const uint32_t key = blk * TC_KB + w * 64 + half * 32 + lane;
        if (blk >= t.hi || key < start || key >= end) return ~0ull;
        const uint32_t slot = key / p.a.page_tokens;
        const uint32_t page = slot < p.kv.table_stride ? __ldg(pages + slot) : 0xFFFFFFFFu;
        if (page >= p.kv.n_pages) {
          bad = 1;
          return ~0ull;
        }
        return page * p.kv.page_stride + (uint64_t)(key - slot * p.a.page_tokens) * p.kv.token_stride + t.kv_head * p.kv.head_stride;
      };
      uint64_t ahead[2] = {look_up(t.lo, 0), look_up(t.lo, 1)};
      bool ok = true;
      for (uint32_t blk = t.lo; blk < t.hi && ok; blk++) {
        const uint64_t place[2] = {ahead[0], ahead[1]};
        ahead[0] = look_up(blk + 1, 0), ahead[1] = look_up(blk + 1, 1);
#pragma unroll 1
        for (int kv = 0; kv < 2; kv++) {
          const T *base = (const T *)(kv ? p.kv.v_pages : p.kv.k_pages);
          if (!(ok = claim(&ctl.empty[stage], phase ^ 1))) break;
          const uint32_t dst = s_ring + stage * S::STAGE;
#pragma unroll
          for (int i = 0; i < (int)(64 * PIECES / 32); i++) {
            const uint32_t idx = i * 32 + lane, r = idx / PIECES, c = idx % PIECES;
            const uint64_t at = __shfl_sync(0xFFFFFFFFu, place[i / (PIECES)], r & 31);
            const bool in = at != ~0ull && c * 8 < D;
            copy16(dst + (c / 8) * (TC_KB * 128) + (w * 64 + r) * 128 + (((c ^ r) & 7) << 4), base + (in ? at + c * 8 : 0), in ? 16 : 0);
          }
          submit(&ctl.full[stage]);
          stage = stage + 1 == S::STAGES ? 0 : stage + 1, phase ^= stage == 0;
        }
      }
      if (!ok) break;
    }
    settle();
    if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
  }
  tm_fence_before();
  __syncthreads();
  if (warp == TC_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512u) : "memory");
}

template <typename T, int DP>
cudaError_t launch_tc(const TcParams &p, int sm_count, cudaStream_t s) {
  const cudaError_t e = cudaFuncSetAttribute(k_attend_tc<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TcShape<DP>::SMEM);
  if (e != cudaSuccess) return e;
  return launch_overlapped(k_attend_tc<T, DP>, dim3(sm_count), TC_THREADS, TcShape<DP>::SMEM, s, false, p);
}
template <typename T>
cudaError_t launch_tc(const TcParams &p, int sm_count, cudaStream_t s) {
  return p.a.head_dim <= 64 ? launch_tc<T, 64>(p, sm_count, s) : launch_tc<T, 128>(p, sm_count, s);
}

}  // namespace

size_t attend_tc_part_floats(int sm_count) { return (size_t)2 * sm_count * part_floats(TC_R, 128); }

cudaError_t launch_attend_tc(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                             int sm_count, cudaStream_t s) {
  const TcParams p{a, kv, q, out, q_stride, out_stride, ws, 2};
  return a.cache_type == MER_VALUE_F16 ? launch_tc<__half>(p, sm_count, s) : launch_tc<__nv_bfloat16>(p, sm_count, s);
}
