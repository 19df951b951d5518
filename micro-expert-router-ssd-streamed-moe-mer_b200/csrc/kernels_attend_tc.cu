// Attention of many new rows over a paged cache: prompts, chunks of prompts, steps that mix them with single tokens.
//
// The same one pass as kernels_attend.cu, on tcgen05: a tile is two groups of 128 rows (tokens x heads of a key head), a block 128 tokens.
//
//   S[128 x 128] = Q[128 x d] K[128 x d]^T      both from shared memory, S in tensor memory
//   P = 2^(S * scale - m + shift)               a thread owns a row: its maximum and sum need no other thread
//   O[128 x d] += P[128 x 128] V[128 x d]       P from tensor memory, where it takes the place of S; V's rows run along N
//
//   * Warps 0..3 and 4..7 are the softmax of one group of rows each, warps 8..11 copy, warp 12 issues the MMAs, warp 13 goes ahead through the run and leaves
//     the next tile's place in shared memory (14 and 15 fill the group).  While one group's
//     softmax runs the tensor core multiplies for the other: [P V of block j, Q K of block j + 1] of one, then of the other.
//   * A tile of up to 128 rows (single tokens, drafts) has one group of rows; the two take its blocks in turn and their results are joined at its end, so that it is
//     read as fast as two groups of rows would be multiplied.
//   * Heads of more than 128 values: a tile has one group of rows, and the two places for scores take its blocks in turn, so that Q K of block j + 1 runs
//     while the first group of warps makes the weights of block j.
//   * The reference maximum of a row follows its maximum only when that has grown by more than 2^LAG; then alone the output in tensor memory is rescaled, by
//     the softmax warps themselves.  Until then weights are larger than 1 by up to that factor, which f16 and fp32 hold.  What makes that safe without a
//     barrier: the MMAs complete in order, so the S of block j being there says that the P V of block j - 1 has been added (with wide heads a barrier says so).
//   * Keys and values come by tiled copies of runs of tokens of a page, 64 values wide; blocks that a sequence's end or a window cuts, and pages that
//     have no such runs (of 1 or 5 tokens, say), row by row, 16 bytes a lane (cp.async), zeros where nothing is to be read.  Row by row alone a
//     block took 4000 cycles in a loop of its own; a prompt of 2048 with pages of one token takes 57 us, 55 with pages of 16.
//   * Rows of P that see nothing of a block hold zeros, and what no row sees is filled with zeros instead of being read.
//   * P is in the cache's type, which the matrix unit wants of both operands: 2^-9 (bf16) or 2^-12 (f16) of each weight at most.  The sums that the output is divided
//     by are of the weights before that, in fp32: their roundings are as often up as down.
// What bounds it: exponentials and MMAs, 2048 cycles each for a block of both groups at 16 and 8192 a cycle; a block takes 3500, the softmax of a group being a
// chain of 2000 between its two MMAs.  32 and 4 heads of 128 in bf16: 2048 rows behind 30700 tokens 970 to 990 us (1.08 PFLOP/s, under the power limit), a
// prompt of 2048 56 us.  Tiles of up to 10 blocks are not cut: prompts of 512, 1024 and 2048 18.6, 26.6 and 55.9 us; cut 24.2, 36.4 and 53.4.
// Every wait is bounded; on expiry the CTA latches MER_DEVSTAT_TIMEOUT, stops issuing work, waits (bounded) for all MMAs and copies that are in
// flight, frees its tensor memory and returns (attend_wait.cuh).
#include <cuda_runtime.h>

#include <algorithm>

#include "attend_join.cuh"
#include "attend_wait.cuh"
#include "attention.cuh"
#include "kernels.h"
#include "pack2.cuh"
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
  uint32_t min_units;
  TileShape ts;
  uint32_t box;  // tokens of a tiled copy, 0: none
  bool head_first;
  bool q_mapped;  // queries by tiled copies
  bool out32;     // output rows are whole pieces of 32 bytes
};
struct TcMaps {
  PageMaps pages;
  CUtensorMap q;  // [row][head][value]
};

constexpr uint32_t TC_KB = 128, TC_WARPS = 16, TC_THREADS = TC_WARPS * 32, SOFT_THREADS = 256;
constexpr uint32_t TC_LOAD = 8, TC_LOADERS = 4, TC_MMA = 12, TC_WALK = 13, TILE_USERS = 13;  // the warps that work on a tile
// Registers of a thread: the launch's 128 times 512 threads, as 192 for the two softmax groups of four warps and 64 for the two others.
constexpr uint32_t SOFT_REGS = 192, OTHER_REGS = 64;
static_assert(2 * SOFT_REGS + 2 * OTHER_REGS == 4 * 128, "what one takes the others give");
// What a tile costs beside its blocks, and a block of two groups of rows, in blocks of one: 8000, 3500 and 1900 cycles (heads of 128; wide heads have tiles of
// one group alone).
constexpr uint32_t TC_START = 4, TC_DENSE = 2, TC_MIN_RUN = 4, TC_WHOLE = 10;
static_assert(TC_MIN_RUN >= TC_DENSE, "every run inside a tile has a block of it");
constexpr float LAG = 7.0f;        // with P_SHIFT the largest weight is 2^15 (scores of a standard deviation of 2: 157 us at 3, 146 so)
constexpr uint32_t TC_CONTROL = 3 * 1024;  // barriers and words in front of the operands, which lie on whole atoms of 1024 bytes

template <int DP>
struct TcShape {
  static constexpr uint32_t SUBS = DP / 64;                // pieces of 64 values of a row
  static constexpr uint32_t STAGE = SUBS * TC_KB * 128;    // keys or values of a block
  static constexpr bool WIDE = DP == 256;                  // one group of rows, whose outputs take as much tensor memory as two groups' of 128 values
  static constexpr uint32_t R = WIDE ? 128 : 256;          // rows of a tile
  static constexpr uint32_t STAGES = DP == 256 ? 2 : DP == 128 ? 5 : 10;
  static constexpr uint32_t QSUB = R * 128;              // 64 values of all queries of a tile
  static constexpr size_t SMEM = TC_CONTROL + SUBS * QSUB + STAGES * STAGE;
};

struct TcControl {
  uint64_t full[10], empty[10];  // stages of the ring
  uint64_t q_full, q_empty, s_full[2], p_half[2], p_ready[2], o_full[2], added, soft, drain;
  uint64_t tile_full[2], tile_empty[2];
  TileWork tile[2];  // tokens == 0: there is none left
  RunStart run;
  RunFound found;
  float one_m[2][128], one_l[2][128];  // what the groups say of rows that both have
  uint32_t tmem, flag[2];  // flags take turns: a sync lies between two uses of one
  volatile uint32_t abort;
};
static_assert(sizeof(TcControl) <= TC_CONTROL && TC_CONTROL % 1024 == 0, "control block");

template <int N>
__device__ __forceinline__ void copies_left() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 bytes to an address on 32 bytes.
__device__ __forceinline__ void store32(void *p, const uint4 &a, const uint4 &b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

template <typename T, int DP>
__global__ void __launch_bounds__(TC_THREADS, 1) k_attend_tc(const TcParams p, const __grid_constant__ TcMaps maps) {
  using S = TcShape<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  TcControl &ctl = *reinterpret_cast<TcControl *>(smem);
  const uint32_t operands = smem_u32(smem) + TC_CONTROL;
  const uint32_t s_q = operands, s_ring = operands + S::SUBS * S::QSUB;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t D = p.a.head_dim, window = p.a.window;
  const TileShape &ts = p.ts;
  if (tid == 0) {
    for (uint32_t i = 0; i < S::STAGES; i++) mbar_init(&ctl.full[i], TC_LOADERS * 32), mbar_init(&ctl.empty[i], 1);
    mbar_init(&ctl.q_full, TC_LOADERS * 32), mbar_init(&ctl.q_empty, 1);
    for (int x = 0; x < 2; x++) mbar_init(&ctl.s_full[x], 1), mbar_init(&ctl.p_half[x], 4), mbar_init(&ctl.p_ready[x], 4), mbar_init(&ctl.o_full[x], 1);
    mbar_init(&ctl.added, 1), mbar_init(&ctl.soft, SOFT_THREADS / 32), mbar_init(&ctl.drain, 1);
    for (int i = 0; i < 2; i++) mbar_init(&ctl.tile_full[i], 1), mbar_init(&ctl.tile_empty[i], TILE_USERS);
    ctl.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == TC_LOAD * 32 && p.box) prefetch_map(&maps.pages.k), prefetch_map(&maps.pages.v);
  if (tid == TC_LOAD * 32 && p.q_mapped) prefetch_map(&maps.q);
  grid_dep_wait();
  grid_dep_launch();
  const RunStart run_here = find_run<TC_KB, TC_THREADS>(p.kv, ts, window, blockIdx.x, gridDim.x, p.min_units, ctl.found);
  if (blockIdx.x == 0) clear_rows_without_place<T, TC_THREADS>(p.a, p.kv, (T *)p.out, p.out_stride, p.ws.status);
  if (blockIdx.x >= run_here.parts) return;
  if (tid == 0) ctl.run = run_here;
  if (warp == TC_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tm = ctl.tmem;
  // columns: S (and P) of the two groups at 0 and 128, their O at 256 and 256 + DP
  auto wait = [&](uint64_t *bar, uint32_t parity) { return wait_or_stop(bar, parity, &ctl.abort, p.ws.status); };
  auto aborted = [&] { return __any_sync(0xFFFFFFFFu, ctl.abort) != 0; };
  // The run's tiles, one after the other; done_with() when the warp no longer looks at one.
  uint32_t turn = 0;
  const RunStart &run = ctl.run;
  auto next_tile = [&] { return wait(&ctl.tile_full[turn & 1], (turn >> 1) & 1) && !aborted() && ctl.tile[turn & 1].tokens != 0; };
  auto done_with = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.tile_empty[turn & 1]);
    turn++;
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFT_REGS));
    // ---------------------------------------------------------------- softmax: a thread has row x * 128 + (tid & 127) of the tile
    const uint32_t x = warp >> 2;
    const uint32_t tm_lane = tm + ((warp & 3) << 21), own_o = tm_lane + 256 + (S::WIDE ? 0 : x * DP);
    const float to_log2 = p.a.scale * LOG2E;
    uint32_t blocks = 0, tiles = 0, syncs = 0, flags = 0;  // phases of s_full, o_full, soft; uses of the flags
    auto sync = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.soft);
      wait(&ctl.soft, syncs++ & 1);
    };
    while (next_tile()) {
      const TileWork &t = ctl.tile[turn & 1];
      const uint32_t rows = t.tokens * t.heads;
      const uint32_t lo = t.lo, hi = t.hi;
      const bool one = S::WIDE || rows <= 128, two_parts = one && !S::WIDE && hi - lo > 1;  // one group of rows, of which both warps' groups have blocks
      const uint32_t row0 = one ? 0 : x * 128, row = row0 + (tid & 127);
      const bool active = S::WIDE ? x == 0 : one ? lo + x < hi : rows > row0;
      const uint32_t tok = min(row, rows - 1) / t.heads, first = t.past + t.token0, see = first + tok;
      const uint32_t least = window && see + 1 > window ? see + 1 - window : 0;  // the row sees least .. see
      float m = -INFINITY, l = 0.0f;
      if (active) {
        // blocks that every row of the group sees whole need no mask
        const uint32_t see0 = first + row0 / t.heads, see1 = first + min(row0 + 127, rows - 1) / t.heads;
        const uint32_t least1 = window && see1 + 1 > window ? see1 + 1 - window : 0;
        const uint32_t blk0 = one ? lo + x : lo;
        for (uint32_t blk = blk0; blk < hi; blk += one && !S::WIDE ? 2 : 1, blocks++) {
          // where the block's scores are, and the phase of that place
          const uint32_t at = S::WIDE ? blocks & 1 : x, phase = S::WIDE ? blocks >> 1 & 1 : blocks & 1, s_at = tm_lane + at * 128;
          if (!wait(&ctl.s_full[at], phase)) break;
          tm_fence_after();
          float s[4][32];
#pragma unroll
          for (int h = 0; h < 4; h++) tm_load_begin(s_at + h * 32, s[h]);
          tm_wait_load();
#pragma unroll
          for (int h = 0; h < 4; h++) tm_loaded(s[h]);
          const uint32_t key0 = blk * TC_KB;
          if (key0 + TC_KB - 1 > see0) {  // the row sees the first `seen` tokens of the block
            const int seen = (int)(see + 1) - (int)key0;
#pragma unroll
            for (int i = 0; i < 128; i++) s[i / 32][i % 32] = i < seen ? s[i / 32][i % 32] : -INFINITY;
          }
          if (key0 < least1) {  // and not the first `old` ones
            const int old = (int)least - (int)key0;
#pragma unroll
            for (int i = 0; i < 128; i++) s[i / 32][i % 32] = i >= old ? s[i / 32][i % 32] : -INFINITY;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 128; i += 8)
#pragma unroll
            for (int e = 0; e < 4; e++) top[e] = fmaxf(fmaxf(s[i / 32][i % 32 + 2 * e], s[i / 32][i % 32 + 2 * e + 1]), top[e]);
          const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * to_log2;
          const bool grow = now > m + LAG || (m == -INFINITY && now > m);
          if (__any_sync(0xFFFFFFFFu, grow)) {
            const float f = grow ? (m == -INFINITY ? 0.0f : exp2_approx(m - now)) : 1.0f;
            if (grow) m = now;
            l *= f;
            if (S::WIDE && blk != blk0 && !wait(&ctl.added, (blocks - 1) & 1)) break;
            if (blk != blk0) {
              if (S::WIDE) tm_fence_after();
              float o[32];
#pragma unroll 1
              for (int c = 0; c < DP; c += 32) {
                tm_load(own_o + c, o);
                uint32_t v[32];
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = __float_as_uint(o[i] * f);
                tm_store(own_o + c, v);
              }
            }
          }
          const float less = m == -INFINITY ? 0.0f : m - P_SHIFT;
          uint64_t sum[2] = {0, 0};
          const uint64_t scale2 = pack2(to_log2, to_log2), less2 = pack2(-less, -less);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
              const uint64_t at = fma2(pack2(s[2 * h + i / 16][2 * i % 32], s[2 * h + i / 16][2 * i % 32 + 1]), scale2, less2);
              float a, b;
              unpack2(at, a, b);
              a = exp2_approx(a), b = exp2_approx(b);
              sum[i & 1] = add2(sum[i & 1], pack2(a, b));
              v[i] = Num<T>::pack(a, b);
            }
            tm_store(s_at + h * 32, v);
            tm_wait_store();
            tm_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(h ? &ctl.p_ready[at] : &ctl.p_half[at]);
          }
          {
            float a, b;
            unpack2(add2(sum[0], sum[1]), a, b);
            l += a + b;
          }
        }
      }
      const bool whole = lo == t.tile_lo && hi == t.tile_hi;
      if (active && !wait(&ctl.o_full[x], tiles++ & 1)) break;
      tm_fence_after();
      // Rows of one group: each group of warps sees to half of their values, of both outputs in tensor memory.
      const bool ends = one || active;
      float f0 = 1.0f, f1 = 0.0f;  // factors of the two outputs
      if (one) {
        ctl.one_m[x][row] = m, ctl.one_l[x][row] = l;
        tm_fence_before();
        sync();
        tm_fence_after();
        const float m0 = ctl.one_m[0][row], m1 = ctl.one_m[1][row];
        m = fmaxf(m0, m1);
        f0 = m0 == -INFINITY ? 0.0f : exp2_approx(m0 - m), f1 = m1 == -INFINITY ? 0.0f : exp2_approx(m1 - m);
        l = ctl.one_l[0][row] * f0 + ctl.one_l[1][row] * f1;
      }
      const int c_first = one && x == 1 ? DP / 2 : 0, c_end = one && x == 0 ? DP / 2 : DP;
      const uint32_t o_at = one ? tm_lane + 256 : own_o;
      auto load_o = [&](int c, float(&o)[32]) {
        __syncwarp();
        tm_load(o_at + c, o);
        if (two_parts) {
          float o1[32];
          tm_load(o_at + DP + c, o1);
#pragma unroll
          for (int i = 0; i < 32; i++) o[i] = o[i] * f0 + o1[i] * f1;
        }
      };
      // The rows of a tile that other runs have parts of.  Its first run comes to it last, at its own end: mostly the others have left their parts by then,
      // and it adds them to what it has.  Where they have not, it leaves its own like them, and whoever arrives last joins them, in the same order.
      uint32_t c0 = 0, n = 1, mine = 0;  // `mine`: this CTA has part 0 and all others are there
      bool joins = whole;
      if (!whole) {
        runs_of_tile(run, t, &c0, &n);
        if (blockIdx.x == c0) {
          if (tid == 0) ctl.flag[flags & 1] = load_acquire(p.ws.counts + c0) == n - 1;
          sync();
          joins = mine = ctl.flag[flags++ & 1];
        }
      }
      // Parts lie as [piece of four values][row]: the rows of a warp side by side.
      if (!joins) {
        float *part = p.ws.parts + (size_t)part_slot(run, t, blockIdx.x) * part_floats(S::R, DP);
        if (ends) {
          if (row < rows && c_first == 0) part[row] = m, part[S::R + row] = l;
#pragma unroll 1
          for (int c = c_first; c < c_end; c += 32) {
            float o[32];
            load_o(c, o);
            if (row < rows) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) reinterpret_cast<float4 *>(part + 2 * S::R)[(c + i) / 4 * S::R + row] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
        }
        sync();
        if (tid == 0) ctl.flag[flags & 1] = arrive_acq_rel(p.ws.counts + c0) + 1 == n;
        sync();
        joins = ctl.flag[flags++ & 1];
      }
      if (!whole && joins && tid == 0) p.ws.counts[c0] = 0;
      if (joins && ends) {
        const bool own = whole || mine;  // part 0 is in tensor memory
        const uint32_t head = t.head0 + min(row, rows - 1) - tok * t.heads;
        // the row's reference and sum over all parts
        const uint32_t k0 = own ? 1 : 0;
        float top = own ? m : -INFINITY, total;
        for (uint32_t k = k0; k < n; k++) top = fmaxf(top, __ldcg(part_of_tile(run, t, p.ws.parts, c0, k, part_floats(S::R, DP)) + row));
        auto weight = [&](float m_of) { return m_of == -INFINITY ? 0.0f : exp2_approx(m_of - top); };
        const float own_f = own ? weight(m) : 0.0f;
        total = l * own_f;
        for (uint32_t k = k0; k < n; k++) {
          const float *from = part_of_tile(run, t, p.ws.parts, c0, k, part_floats(S::R, DP)) + row;
          total = k == 0 ? weight(__ldcg(from)) * __ldcg(from + S::R) : fmaf(weight(__ldcg(from)), __ldcg(from + S::R), total);
        }
        if (p.a.sinks) total += sink_weight(p.a.sinks, head, top);
        const float f = total == 0.0f ? 0.0f : 1.0f / total;
        T *out = (T *)p.out + (uint64_t)(t.row0 + t.token0 + tok) * p.out_stride + (uint64_t)head * D;
#pragma unroll 1
        for (int c = c_first; c < c_end; c += 32) {
          float o[32];
          load_o(c, o);
#pragma unroll
          for (int i = 0; i < 32; i++) o[i] *= own_f;
          for (uint32_t k = k0; k < n; k++) {
            const float *from = part_of_tile(run, t, p.ws.parts, c0, k, part_floats(S::R, DP));
            float4 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __ldcg(reinterpret_cast<const float4 *>(from + 2 * S::R) + (c / 4 + i) * S::R + row);
            const float w = weight(__ldcg(from + row));
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const bool start = k == 0;
              o[4 * i] = start ? w * v[i].x : fmaf(w, v[i].x, o[4 * i]), o[4 * i + 1] = start ? w * v[i].y : fmaf(w, v[i].y, o[4 * i + 1]);
              o[4 * i + 2] = start ? w * v[i].z : fmaf(w, v[i].z, o[4 * i + 2]), o[4 * i + 3] = start ? w * v[i].w : fmaf(w, v[i].w, o[4 * i + 3]);
            }
          }
          if (row >= rows) continue;
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; i++)
            v[i] = make_uint4(Num<T>::pack(o[8 * i] * f, o[8 * i + 1] * f), Num<T>::pack(o[8 * i + 2] * f, o[8 * i + 3] * f), Num<T>::pack(o[8 * i + 4] * f, o[8 * i + 5] * f),
                              Num<T>::pack(o[8 * i + 6] * f, o[8 * i + 7] * f));
          if (p.out32) {  // a lane's rows lie apart: the wider its stores, the fewer lines they touch
            if (c < (int)D) store32(out + c, v[0], v[1]);
            if (c + 16 < (int)D) store32(out + c + 16, v[2], v[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (c + 8 * i < (int)D) *reinterpret_cast<uint4 *>(out + c + 8 * i) = v[i];
          }
        }
      }
      tm_fence_before();
      if (one) sync();  // both outputs have been read
      done_with();
    }
  } else if (warp >= TC_MMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == TC_MMA) {
    // ---------------------------------------------------------------- MMA issue
    const uint32_t leader = tm_elect();
    constexpr uint32_t TYPE = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t BASE = (1u << 4) | (TYPE << 7) | (TYPE << 10) | ((128u >> 4) << 24);
    constexpr uint32_t QK = BASE | ((TC_KB >> 3) << 17), PV = BASE | (1u << 16) | ((DP >> 3) << 17);
    uint32_t tiles = 0, blocks0 = 0, blocks1 = 0, at = 0, turns = 0;  // phases of q_full and p_ready; places of the ring before the tile's: keys of its block j are at + 2 j, values the next
    auto place = [&](uint64_t *bars, uint32_t q) { return &bars[q % S::STAGES]; };
    auto landed = [&](uint32_t q) { return wait(place(ctl.full, q), (q / S::STAGES) & 1); };
    // Descriptors of rows of 128 bytes in atoms of 8 rows (1024 bytes), 128-byte swizzle.  Bits: start >> 4 [0,14), leading offset >> 4 [16,30), stride offset >> 4
    // [32,46), version 1 [46,48), swizzle 2 [61,64).  An operand whose rows run along K: 1024 between atoms, no leading offset; one whose rows run along N: 1024
    // between groups of 8 of K, the leading offset between pieces of 64 values of a row.  The starts of an operand's pieces lie constants apart.
    constexpr uint64_t ALONG_K = (64ull << 32) | (1ull << 46) | (2ull << 61) | (1ull << 16), ALONG_N = (64ull << 32) | (1ull << 46) | (2ull << 61) | ((uint64_t)(TC_KB * 128 >> 4) << 16);
    const uint32_t q_at = s_q >> 4, ring_at = s_ring >> 4;
    auto qk = [&](uint32_t x, uint32_t rows_of, uint32_t q) {  // the scores of a group for the keys at place q
      const uint32_t a = q_at + rows_of * (16384 >> 4), b = ring_at + q % S::STAGES * (S::STAGE >> 4);
#pragma unroll
      for (int k = 0; k < DP / 16; k++)
        tm_mma_ss(leader, tm + x * 128, ALONG_K | (a + (k / 4) * (S::QSUB >> 4) + (k & 3) * 2), ALONG_K | (b + (k / 4) * (TC_KB * 128 >> 4) + (k & 3) * 2), QK, k != 0);
      tm_commit(leader, &ctl.s_full[x]);
    };
    auto pv = [&](uint32_t x, uint32_t q, bool first) {  // its weights (of place x) times the values at place q
      const uint32_t b = ring_at + q % S::STAGES * (S::STAGE >> 4);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (!wait(h ? &ctl.p_ready[x] : &ctl.p_half[x], (x ? blocks1 : blocks0) & 1)) return false;
        tm_fence_after();
#pragma unroll
        for (int k = 4 * h; k < 4 * h + 4; k++) tm_mma_ts(leader, tm + 256 + (S::WIDE ? 0 : x * DP), tm + x * 128 + k * 8, ALONG_N | (b + k * 128), PV, k != 0 || !first);
      }
      blocks0 += x == 0, blocks1 += x == 1;
      return true;
    };
    auto free_place = [&](uint32_t q) { tm_commit(leader, place(ctl.empty, q)); };
    while (next_tile()) {
      const TileWork &t = ctl.tile[turn & 1];
      const uint32_t rows = t.tokens * t.heads, lo = t.lo, n = t.hi - t.lo;
      // Blocks below `by_rows` and from `by_rows_again` on are filled row by row: not by the proxy that the tensor core reads through.
      const uint32_t by_rows = p.box ? (first_seen(t, window) + TC_KB - 1) / TC_KB : 0xFFFFFFFFu, by_rows_again = (t.past + t.token0 + t.tokens) / TC_KB;
      auto visible = [&](uint32_t j) {
        if (lo + j < by_rows || lo + j >= by_rows_again) proxy_fence();
      };
      done_with();
      if (!wait(&ctl.q_full, tiles++ & 1)) break;
      if (!p.q_mapped) proxy_fence();
      bool ok = true;
      if (S::WIDE) {  // the places for scores take the blocks in turn
        for (uint32_t j = 0; j <= n && ok; j++) {
          if (j < n) {
            if (!(ok = landed(at + 2 * j))) break;
            visible(j);
            tm_fence_after();
            qk((turns + j) & 1, 0, at + 2 * j);
            free_place(at + 2 * j);
            if (j + 1 == n) tm_commit(leader, &ctl.q_empty);
          }
          if (j == 0) continue;
          const uint32_t v = at + 2 * j - 1;
          if (!(ok = landed(v))) break;
          visible(j - 1);
          if (!(ok = pv((turns + j - 1) & 1, v, j == 1))) break;
          free_place(v);
          tm_commit(leader, &ctl.added);
          if (j == n) tm_commit(leader, &ctl.o_full[0]);
        }
        turns += n;
      } else if (rows <= 128) {  // the groups take the blocks in turn
        for (uint32_t j = 0; j < 2 && j < n && ok; j++) {
          if (!(ok = landed(at + 2 * j))) break;
          visible(j);
          tm_fence_after();
          qk(j, 0, at + 2 * j);
          free_place(at + 2 * j);
          if (j + 1 == n) tm_commit(leader, &ctl.q_empty);
        }
        for (uint32_t j = 0; j < n && ok; j++) {
          const uint32_t x = j & 1, v = at + 2 * j + 1, k = at + 2 * (j + 2);
          if (!(ok = landed(v))) break;
          visible(j);
          if (!(ok = pv(x, v, j < 2))) break;
          free_place(v);
          if (j + 2 < n) {
            if (!(ok = landed(k))) break;
            visible(j + 2);
            qk(x, 0, k);
            free_place(k);
            if (j + 3 == n) tm_commit(leader, &ctl.q_empty);
          } else {
            tm_commit(leader, &ctl.o_full[x]);
          }
        }
      } else {
        if (!landed(at)) break;
        visible(0);
        tm_fence_after();
        for (uint32_t x = 0; x < 2; x++) qk(x, x, at);
        free_place(at);
        if (n == 1) tm_commit(leader, &ctl.q_empty);
        for (uint32_t j = 0; j < n && ok; j++) {
          const uint32_t v = at + 2 * j + 1, k = v + 1;
          const bool more = j + 1 < n;
          if (!(ok = landed(v))) break;
          if (more && !(ok = landed(k))) break;
          visible(j);
          if (more) visible(j + 1);
          for (uint32_t x = 0; x < 2; x++) {
            if (!(ok = pv(x, v, j == 0))) break;
            if (more)
              qk(x, x, k);
            else
              tm_commit(leader, &ctl.o_full[x]);
          }
          if (!ok) break;
          free_place(v);
          if (more) {
            free_place(k);
            if (j + 2 == n) tm_commit(leader, &ctl.q_empty);
          }
        }
      }
      if (!ok) break;
      at += 2 * n;
    }
    } else if (warp == TC_WALK) {
      // -------------------------------------------------------------- the way through the run
      RunWalk<TC_KB> walk(p.kv, ts, window, ctl.run);
      TileWork t;
      for (uint32_t i = 0;; i++) {
        const bool more = walk.next(&t);
        if (!more) t.tokens = 0;
        if (!wait(&ctl.tile_empty[i & 1], ((i >> 1) & 1) ^ 1)) break;
        if (lane == 0) {
          ctl.tile[i & 1] = t;
          mbar_arrive(&ctl.tile_full[i & 1]);
        }
        if (!more) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    // ---------------------------------------------------------------- copies: warp w has the rows w * 32 .. of a block, and a quarter of the queries
    const uint32_t w = warp - TC_LOAD;
    uint32_t stage = 0, phase = 0, tiles = 0, bad = 0;
    // The barrier counts a lane's copies when they have landed; the MMA warp makes them visible to the tensor core.  (A proxy fence
    // here would wait for the copies behind them as well: 4900 cycles a block, 2 stages in flight instead of 5.)
    auto submit = [&](uint64_t *bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); };
    // 32 rows from shared-memory address `dst` on; a lane has the place of one of them in pieces of 16 bytes, ~0: zeros.  Lane i copies piece
    // i % PIECES of every row that it has a part in, whose place in the swizzle repeats after 8 rows.
    constexpr uint32_t PIECES = DP / 8, AT_ONCE = 32 / PIECES;  // pieces of a row, rows of one instruction
    const uint32_t c = lane % PIECES, r0 = lane / PIECES;
    const uint32_t col = c & 7;
    const bool in_head = c * 8 < D;
    auto copy_rows = [&](uint32_t dst, uint32_t sub, const void *base, uint32_t place) {
      const char *from = (const char *)base + c * 16;
      dst += (c / 8) * sub + r0 * 128;
#pragma unroll
      for (uint32_t i = 0; i < 32 / AT_ONCE; i++) {
        const uint32_t r = i * AT_ONCE + r0, at = __shfl_sync(0xFFFFFFFFu, place, r);
        const bool in = at != 0xFFFFFFFFu && in_head;
        copy16(dst + i * (AT_ONCE * 128) + ((col ^ (r & 7)) << 4), in ? from + (uint64_t)at * 16 : (const char *)base, in ? 16 : 0);
      }
    };
    while (next_tile()) {
      const TileWork t = ctl.tile[turn & 1];
      done_with();
      const uint32_t rows = t.tokens * t.heads;
      if (!wait(&ctl.q_empty, (tiles & 1) ^ 1)) break;
      if (p.q_mapped) {
        // 64 values of ts.heads heads of ts.tokens rows; those behind the sequence's end are other rows or zeros, which nobody stores
        if (lane == 0 && w < S::SUBS) {
          const uint32_t bar = smem_u32(&ctl.q_full);
          mbar_expect_tx(&ctl.q_full, ts.tokens * ts.heads * 128);
          asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(s_q + w * S::QSUB),
                       "l"(&maps.q), "r"(w * 64), "r"(t.head0), "r"(t.row0 + t.token0), "r"(bar)
                       : "memory");
        } else {
          mbar_arrive(&ctl.q_full);
        }
      } else {
#pragma unroll 1
        for (uint32_t i = 0; i < S::R / (TC_LOADERS * 32); i++) {
          const uint32_t r = w * (S::R / TC_LOADERS) + i * 32 + lane, tok = r / t.heads;
          // the tile's rows lie within 2^32 pieces of its first one
          const uint32_t place = r < rows ? tok * (uint32_t)(p.q_stride / 8) + (r - tok * t.heads) * (D / 8) : 0xFFFFFFFFu;
          copy_rows(s_q + (w * (S::R / TC_LOADERS) + i * 32) * 128, S::QSUB, (const T *)p.q + (uint64_t)(t.row0 + t.token0) * p.q_stride + t.head0 * D, place);
        }
        submit(&ctl.q_full);
      }
      tiles++;
      const uint32_t end = t.past + t.token0 + t.tokens;
      const uint32_t start = first_seen(t, window);
      const PagePlaces pages(p.kv, p.a.page_tokens, t.seq, t.kv_head);
      // a lane's token of a block: the first of its tiled copy, or a row
      constexpr uint32_t SUBS = S::SUBS;
      const uint32_t copy = lane * TC_LOADERS + w, copy_row = copy / SUBS * p.box, copies = p.box ? TC_KB / p.box * SUBS : 0;
      auto tiled = [&](uint32_t blk) { return p.box && blk * TC_KB >= start && blk * TC_KB + TC_KB <= end; };
      auto entry = [&](uint32_t blk) {
        const bool whole = tiled(blk);
        const uint32_t key = blk * TC_KB + (whole ? copy_row : w * 32 + lane);
        return blk < t.hi && (whole ? copy < copies : key >= start && key < end) ? pages.entry(key) : 0u;
      };
      uint32_t ahead[2] = {entry(t.lo), entry(t.lo + 1)};
      bool ok = true;
      for (uint32_t blk = t.lo; blk < t.hi && ok; blk++) {
        const uint32_t number = ahead[0];
        ahead[0] = ahead[1];
        ahead[1] = entry(blk + 2);
        if (tiled(blk)) {
          const uint32_t token = pages.in_page(blk * TC_KB + copy_row);
          if (copy < copies && number >= p.kv.n_pages) bad = 1;
#pragma unroll 1
          for (int kv = 0; kv < 2; kv++) {
            if (!(ok = wait(&ctl.empty[stage], phase ^ 1))) break;
            if (copy < copies) {
              mbar_expect_tx(&ctl.full[stage], p.box * 128);
              page_g2s(s_ring + stage * S::STAGE + (copy % SUBS) * (TC_KB * 128) + copy_row * 128, kv ? &maps.pages.v : &maps.pages.k, (copy % SUBS) * 64, token, t.kv_head,
                       min(number, p.kv.n_pages), p.head_first, smem_u32(&ctl.full[stage]));
            } else {
              mbar_arrive(&ctl.full[stage]);
            }
            stage = stage + 1 == S::STAGES ? 0 : stage + 1, phase ^= stage == 0;
          }
        } else {
          const uint32_t key = blk * TC_KB + w * 32 + lane;
          const uint32_t place = key >= start && key < end ? pages.place(key, number, &bad) : 0xFFFFFFFFu;
#pragma unroll 1
          for (int kv = 0; kv < 2; kv++) {
            if (!(ok = wait(&ctl.empty[stage], phase ^ 1))) break;
            copy_rows(s_ring + stage * S::STAGE + w * (32 * 128), TC_KB * 128, kv ? p.kv.v_pages : p.kv.k_pages, place);
            submit(&ctl.full[stage]);
            stage = stage + 1 == S::STAGES ? 0 : stage + 1, phase ^= stage == 0;
          }
        }
      }
      if (!ok) break;
    }
    copies_left<0>();
    if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
  }
  tm_fence_before();
  __syncthreads();
  // After a wait that has run out: MMAs, and tiled copies of keys, values and queries.  Only here is it certain that no warp gives up any more: those that
  // issued them may have ended long before.
  const bool gave_up = ctl.abort != 0;
  if (warp == TC_MMA) {
    if (gave_up) {
      tm_commit(tm_elect(), &ctl.drain);  // the lane that issued: the same one is elected every time
      mbar_drain(&ctl.drain, 0, 1000000000ull);
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512u) : "memory");
  }
  if (gave_up && tid <= S::STAGES) drain_copies(tid < S::STAGES ? &ctl.full[tid] : &ctl.q_full);
}

template <typename T, int DP>
cudaError_t launch_tc(const TcParams &p, const TcMaps &maps, int sm_count, cudaStream_t s) {
  const cudaError_t e = allow_smem<k_attend_tc<T, DP>>(TcShape<DP>::SMEM);
  if (e != cudaSuccess) return e;
  return launch_overlapped(k_attend_tc<T, DP>, dim3(sm_count), TC_THREADS, TcShape<DP>::SMEM, s, false, p, maps);
}
template <typename T>
cudaError_t launch_tc(const TcParams &p, const TcMaps &maps, int sm_count, cudaStream_t s) {
  if (p.a.head_dim <= 64) return launch_tc<T, 64>(p, maps, sm_count, s);
  return p.a.head_dim <= 128 ? launch_tc<T, 128>(p, maps, sm_count, s) : launch_tc<T, 256>(p, maps, sm_count, s);
}

}  // namespace

size_t attend_tc_part_floats(int sm_count) { return (size_t)2 * sm_count * std::max(part_floats(TcShape<128>::R, 128), part_floats(TcShape<256>::R, 256)); }

cudaError_t launch_attend_tc(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                             int sm_count, cudaStream_t s) {
  const PageMapShape m(a, kv, TC_KB);
  TcMaps maps{};
  const bool mapped = encode_page_maps(&maps.pages, m, a, kv);
  TcParams p{a, kv, q, out, q_stride, out_stride, ws, TC_MIN_RUN, TileShape(a.q_heads, a.kv_heads, a.head_dim <= 128 ? TcShape<128>::R : TcShape<256>::R, TC_START, TC_DENSE, a.head_dim <= 128 ? 128 : 0xFFFFFFFFu, TC_WHOLE), mapped ? m.rows : 0, m.head_first, false, false};
  p.q_mapped = p.ts.chunks == 1 && encode_row_map(&maps.q, q, a, kv.n_rows, q_stride, p.ts.heads, p.ts.tokens);
  p.out32 = a.head_dim % 16 == 0 && ((uintptr_t)out | out_stride * 2) % 32 == 0;
  return a.cache_type == MER_VALUE_F16 ? launch_tc<__half>(p, maps, sm_count, s) : launch_tc<__nv_bfloat16>(p, maps, sm_count, s);
}
