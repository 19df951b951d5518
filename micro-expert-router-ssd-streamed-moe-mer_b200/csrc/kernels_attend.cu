// Attention of single new tokens over a paged cache.  Head sizes up to 256 in steps of 8.
//
//   o = sum_j 2^(s_j - m) v_j / (sum_j 2^(s_j - m) [+ 2^(sink - m)]),  s_j = q . k_j * scale * log2 e,  m = max_j s_j
//
// in one pass over the keys with the running maximum and sum of every row.  What bounds it is reading the cache: per 16 tokens 16 * 2 *
// head_dim values for at most 16 rows of work.  So a warp is a stream of its own: it copies the next chunks of 16 tokens (tiled copies of 8 or 16
// tokens of a page; row by row, 16 bytes a lane, where a sequence's end or a window cuts a chunk or pages have no such runs) into a ring that no other warp sees, multiplies the one that has landed (mma.sync on 16 x 16 tiles; at this rate of
// operations the legacy tensor path is idle most of the time) and keeps maximum, sum and output of its own tokens in registers: no barrier
// in the loop.  The warps' results are joined in shared memory at the end of a tile, those of several CTAs through the workspace (attention.cuh).
// 64 tokens behind 800 to 8000 (32 and 4 heads of 128, bf16) 81 to 87 us by the box, 5.4 to 5.8 TB/s; one behind 32000 22 us, of which 10 are reading and the rest the
// dependent reads at the run's beginning and the join at its end.  Pages of one token, copied row by row: 84 us for the 64 tokens, 81 with pages of 16 on the same box.  Tiles of up to 4 blocks are not cut: 16 windows of 128 tokens 7.0 us, 8.9 cut.
// The weights go to the second product in the cache's type, 2^-9 (bf16) or 2^-12 (f16) of each at most, like the values they multiply; sums are fp32.
// Every wait is bounded; one that runs out is latched as MER_DEVSTAT_TIMEOUT and stops the CTA (attend_wait.cuh).
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"
#include "attend_join.cuh"
#include "attend_wait.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace {

constexpr uint32_t WHOLE_BLOCKS = 4;  // of a tile that is not cut
constexpr uint32_t START_UNITS = 3;  // what a tile costs beside its blocks, in blocks

struct AttendParams {
  AttnLayer a;
  KvBatchDev kv;
  const void *q;
  void *out;
  uint64_t q_stride, out_stride;
  AttnWorkspace ws;
  TileShape ts;
  uint32_t box;  // tokens of a tiled copy (8 or 16), 0: none
  bool head_first;
};

// Warps NW, chunks in flight per warp ST.
template <int DP>
struct StreamShape {
  static constexpr int NW = DP == 256 ? 4 : 8, ST = DP == 64 ? 6 : 3;
  static constexpr uint32_t KB = NW * 16, THREADS = NW * 32, CHUNK = 2 * 16 * DP * 2;
};

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4_trans(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// A load that stays where it stands among the copies.  An ordinary one: the kernel in front, which writes the queries, may still run when this one starts.
__device__ __forceinline__ uint4 load_now(const void *p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
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

// Byte offset of 16-byte piece `c` of row `r` of ROWS: 64 values of every row, then the next 64, in the 128-byte swizzle; eight rows of one
// column of pieces lie in eight different bank groups.
template <uint32_t ROWS>
__device__ __forceinline__ uint32_t piece(uint32_t r, uint32_t c) {
  return (c >> 3) * (ROWS * 128) + r * 128 + (((c ^ r) & 7) << 4);
}

template <typename T, int DP>
__global__ void __launch_bounds__(StreamShape<DP>::THREADS, 1) k_attend_stream(const AttendParams p, const __grid_constant__ PageMaps maps) {
  using S = StreamShape<DP>;
  constexpr int NW = S::NW, ST = S::ST, R = 16;
  constexpr uint32_t KB = S::KB, THREADS = S::THREADS;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ uint64_t s_full[NW * ST];  // a chunk has landed: every lane of its warp arrives
  __shared__ RunFound s_found;
  __shared__ uint32_t s_flag;
  __shared__ volatile uint32_t s_stop;  // a wait has run out
  __shared__ uint64_t s_join;
  uint8_t *s_ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);  // [NW][ST][k, v][DP / 64][16][64]
  uint8_t *s_q = s_ring + NW * ST * S::CHUNK;                                  // [DP / 64][R][64]
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t D = p.a.head_dim, page_tokens = p.a.page_tokens, window = p.a.window;
  const TileShape &ts = p.ts;
  for (uint32_t i = tid; i < NW * ST; i += THREADS) mbar_init(&s_full[i], 32);
  if (tid == 0) mbar_init(&s_join, 1), s_stop = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (tid == 0 && p.box) prefetch_map(&maps.k), prefetch_map(&maps.v);
  grid_dep_wait();
  grid_dep_launch();
  const RunStart run = find_run<KB, THREADS>(p.kv, ts, window, blockIdx.x, gridDim.x, 1, s_found);
  if (blockIdx.x == 0) clear_rows_without_place<T, THREADS>(p.a, p.kv, (T *)p.out, p.out_stride, p.ws.status);
  if (blockIdx.x >= run.parts) return;
  RunWalk<KB> walk(p.kv, ts, window, run);
  const float to_log2 = p.a.scale * LOG2E;
  uint32_t fill = 0, stage = 0, stage_phase = 0, join_phase = 0;  // of the warp's ring: what is asked for next, what is taken next
  bool chunk_lost = false, join_lost = false;  // the warp has given up the wait for a chunk, or for parts
  const uint32_t ring = smem_u32(s_ring) + warp * (ST * S::CHUNK), q_addr = smem_u32(s_q);

  TileWork t;
  while (walk.next(&t)) {
    const uint32_t rows = t.tokens * t.heads;
    const uint32_t end = t.past + t.token0 + t.tokens;  // behind the last token that a row of the tile sees
    const uint32_t start = first_seen(t, window);
    // ---- the ring.  A lane knows where its part of a chunk lies, ST chunks ahead: lanes 0 .. 15 a row of one that is copied row by row; of others, the first
    // lanes a tiled copy of the keys each, the next ones of the values.
    const PagePlaces pages(p.kv, page_tokens, t.seq, t.kv_head);
    constexpr uint32_t SUBS = DP / 64;
    const uint32_t copies = p.box ? 16 / p.box * SUBS : 0, copy = lane < copies ? lane : lane - copies, copy_row = copy / SUBS * p.box;
    uint32_t bad = 0;
    auto wanted = [&](uint32_t blk) { return blk < t.hi && blk * KB + warp * 16 < end && blk * KB + warp * 16 + 16 > start; };
    auto tiled = [&](uint32_t blk) { return p.box && blk * KB + warp * 16 >= start && blk * KB + warp * 16 + 16 <= end; };
    auto key_of = [&](uint32_t blk) { return blk * KB + warp * 16 + (tiled(blk) ? copy_row : lane & 15); };
    auto to_read = [&](uint32_t blk) { return wanted(blk) && (tiled(blk) ? lane < 2 * copies : key_of(blk) >= start && key_of(blk) < end); };
    auto entry = [&](uint32_t blk) { return to_read(blk) ? pages.entry(key_of(blk)) : 0u; };
    auto issue = [&](uint32_t blk, uint32_t number) {
      if (!wanted(blk)) return;
      const uint32_t dst = ring + fill * S::CHUNK, bar = smem_u32(&s_full[warp * ST + fill]);
      fill = fill + 1 == ST ? 0 : fill + 1;
      if (tiled(blk)) {
        if (start) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage may have been filled row by row
        if (lane < 2 * copies) {
          if (number >= p.kv.n_pages) bad = 1;
          const bool v = lane >= copies;
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(p.box * 128) : "memory");
          page_g2s(dst + (v ? 16 * DP * 2 : 0) + (copy % SUBS) * 2048 + copy_row * 128, v ? &maps.v : &maps.k, (copy % SUBS) * 64, pages.in_page(key_of(blk)), t.kv_head,
                   min(number, p.kv.n_pages), p.head_first, bar);
        } else {
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
        }
        return;
      }
      const uint32_t place = to_read(blk) ? pages.place(key_of(blk), number, &bad) : 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < DP / 16; i++) {
        const uint32_t idx = i * 32 + lane, r = idx / (DP / 8), c = idx % (DP / 8);
        const uint32_t at = __shfl_sync(0xFFFFFFFFu, place, r);
        const bool in = at != 0xFFFFFFFFu && c * 8 < D;
        const uint64_t off = in ? ((uint64_t)at + c) * 16 : 0;
        copy16(dst + piece<16>(r, c), (const char *)p.kv.k_pages + off, in ? 16 : 0);
        copy16(dst + 16 * DP * 2 + piece<16>(r, c), (const char *)p.kv.v_pages + off, in ? 16 : 0);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    };
    // Queries are asked for ahead of the keys: behind these they would wait for a full ring of every SM.
    constexpr uint32_t Q_PIECES = (R * (DP / 8) + THREADS - 1) / THREADS;  // of a thread
    uint32_t ahead[ST];
#pragma unroll
    for (int i = 0; i < ST; i++) ahead[i] = entry(t.lo + i);
    uint4 q[Q_PIECES];
#pragma unroll
    for (uint32_t u = 0; u < Q_PIECES; u++) {
      const uint32_t i = tid + u * THREADS, r = i / (DP / 8), c = i % (DP / 8), tok = r / t.heads, h = r - tok * t.heads;
      q[u] = make_uint4(0, 0, 0, 0);
      if (r < rows && c * 8 < D)  // rows <= R: also the threads that have none
        q[u] = load_now((const T *)p.q + (uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + h) * D + c * 8);
    }
#pragma unroll
    for (int i = 0; i < ST - 1; i++) issue(t.lo + i, ahead[i]);
    uint32_t next_entry = ahead[ST - 1];
#pragma unroll
    for (uint32_t u = 0; u < Q_PIECES; u++) {
      const uint32_t i = tid + u * THREADS;
      if (i < R * (DP / 8)) *reinterpret_cast<uint4 *>(s_q + piece<R>(i / (DP / 8), i % (DP / 8))) = q[u];
    }
    __syncthreads();
    // the last tokens that the lane's two rows see
    const uint32_t last[2] = {t.past + t.token0 + min(lane / 4, rows - 1) / t.heads, t.past + t.token0 + min(8 + lane / 4, rows - 1) / t.heads};
    float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < DP / 8; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[i][e] = 0.0f;
    for (uint32_t blk = t.lo; blk < t.hi; blk++) {
      {
        const uint32_t number = next_entry;
        next_entry = entry(blk + ST);
        __syncwarp();  // the chunk that lay in this stage has been read
        issue(blk + ST - 1, number);
      }
      if (!wanted(blk)) continue;
      const uint32_t key0 = blk * KB + warp * 16, base = ring + stage * S::CHUNK;
      if (!wait_or_stop(&s_full[warp * ST + stage], stage_phase, &s_stop, p.ws.status)) {
        chunk_lost = true;
        break;
      }
      stage = stage + 1 == ST ? 0 : stage + 1, stage_phase ^= stage == 0;
      float s[2][4];
      {
        // the products of even and odd pieces of a head apart, so that half as many wait for one another
        float c[2][2][4] = {};
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) {
          uint32_t kf[4], qf[4];
          ldm4(kf, base + piece<16>((lane / 16) * 8 + (lane & 7), kk * 2 + ((lane >> 3) & 1)));
          ldm4(qf, q_addr + piece<R>(((lane >> 3) & 1) * 8 + (lane & 7), kk * 2 + (lane >> 4)));
          mma16816<T>(c[kk & 1][0], qf, kf[0], kf[1]);
          mma16816<T>(c[kk & 1][1], qf, kf[2], kf[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[n][e] = c[0][n][e] + c[1][n][e];
      }
      float top[2] = {-INFINITY, -INFINITY}, less[2];
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t at = key0 + (lane & 3) * 2 + n * 8 + (e & 1), see = last[e >> 1];
          const bool seen = at <= see && (window == 0 || at + window > see);
          s[n][e] = seen ? s[n][e] * to_log2 : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xFFFFFFFFu, top[e], 1));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xFFFFFFFFu, top[e], 2));
        top[e] = fmaxf(top[e], m[e]);
        less[e] = top[e] == -INFINITY ? 0.0f : top[e] - P_SHIFT;
      }
      if (__any_sync(0xFFFFFFFFu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float f = m[e] == -INFINITY ? 0.0f : exp2_approx(m[e] - top[e]);
          l[e] *= f;
          m[e] = top[e];
#pragma unroll
          for (int i = 0; i < DP / 8; i++) o[i][2 * e] *= f, o[i][2 * e + 1] *= f;
        }
      }
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s[n][e] = exp2_approx(s[n][e] - less[e >> 1]);
          l[e >> 1] += s[n][e];
        }
      const uint32_t pf[4] = {Num<T>::pack(s[0][0], s[0][1]), Num<T>::pack(s[0][2], s[0][3]), Num<T>::pack(s[1][0], s[1][1]), Num<T>::pack(s[1][2], s[1][3])};
      const uint32_t vbase = base + 16 * DP * 2;
#pragma unroll
      for (int dn = 0; dn < DP / 16; dn++) {
        uint32_t vf[4];
        ldm4_trans(vf, vbase + piece<16>(((lane >> 3) & 1) * 8 + (lane & 7), dn * 2 + (lane >> 4)));
        mma16816<T>(o[2 * dn], pf, vf[0], vf[1]);
        mma16816<T>(o[2 * dn + 1], pf, vf[2], vf[3]);
      }
    }
    if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
    // ---- the warps' results: [warp][row] maximum and sum, [warp][row][DP] output, where the rings were
    constexpr int OP = DP + 8;  // floats of a row of it: the rows of a fragment lie in different banks
    float *s_m = reinterpret_cast<float *>(s_ring), *s_l = s_m + NW * R, *s_o = s_l + NW * R;
    if (__syncthreads_or(chunk_lost)) break;  // copies may still land in the rings
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float sum = l[e];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      const uint32_t r = e * 8 + lane / 4;
      if (r >= rows) continue;
      if ((lane & 3) == 0) s_m[warp * R + r] = m[e], s_l[warp * R + r] = sum;
#pragma unroll
      for (int i = 0; i < DP / 8; i++) *reinterpret_cast<float2 *>(s_o + ((size_t)warp * R + r) * OP + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
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
        const float4 v = *reinterpret_cast<const float4 *>(s_o + ((size_t)w * R + r) * OP + c);
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
    if (!whole) {
      __syncthreads();
      // The CTA that arrives last joins the parts in the order of the runs and leaves the count at zero.  A part's maxima, sums and rows lie one behind the
      // other: each is one bulk copy into the rings, all in flight at once (a round trip for what other SMs have just written is 1500 to 3000 cycles).
      uint32_t c0, n;
      runs_of_tile(run, t, &c0, &n);
      if (tid == 0) {
        const bool is_last = arrive_acq_rel(p.ws.counts + c0) + 1 == n;
        if (is_last) p.ws.counts[c0] = 0;
        s_flag = is_last;
      }
      asm volatile("fence.proxy.async;" ::: "memory");  // what this CTA has in the rings, and what the others have left in memory
      __syncthreads();
      if (s_flag) {
        constexpr int V = DP / 32, TURNS = R / NW;  // values of a lane, rows of a warp
        const uint32_t each = 2 * R + rows * DP, at_once = NW * ST * S::CHUNK / 4 / each;
        const float *s_parts = reinterpret_cast<const float *>(s_ring);
        float acc[TURNS][V], top[TURNS], total[TURNS];
#pragma unroll
        for (int u = 0; u < TURNS; u++) {
          top[u] = -INFINITY, total[u] = 0.0f;
#pragma unroll
          for (int i = 0; i < V; i++) acc[u][i] = 0.0f;
        }
        for (uint32_t k0 = 0; k0 < n; k0 += at_once) {
          const uint32_t some = min(at_once, n - k0);
          asm volatile("fence.proxy.async;" ::: "memory");
          if (__syncthreads_or(join_lost)) break;
          if (tid == 0) mbar_expect_tx(&s_join, some * each * 4);
          for (uint32_t k = tid; k < some; k += THREADS)
            bulk_g2s(s_ring + (size_t)k * each * 4, part_of_tile(run, t, p.ws.parts, c0, k0 + k, part_floats(R, DP)), each * 4, &s_join);
          join_lost = !wait_or_stop(&s_join, join_phase, &s_stop, p.ws.status);
          join_phase ^= 1;
#pragma unroll
          for (int u = 0; u < TURNS; u++) {
            const uint32_t r = warp + u * NW;
            if (r >= rows) continue;
            float now = top[u];
            for (uint32_t k = lane; k < some; k += 32) now = fmaxf(now, s_parts[k * each + r]);
#pragma unroll
            for (int d = 16; d; d /= 2) now = fmaxf(now, __shfl_xor_sync(0xFFFFFFFFu, now, d));
            const float old = top[u] == -INFINITY ? 0.0f : exp2_approx(top[u] - now);
            top[u] = now;
            total[u] *= old;
#pragma unroll
            for (int i = 0; i < V; i++) acc[u][i] *= old;
#pragma unroll 4
            for (uint32_t k = 0; k < some; k++) {
              const float *part = s_parts + k * each;
              const float m = part[r], f = m == -INFINITY ? 0.0f : exp2_approx(m - now);
              total[u] = fmaf(f, part[R + r], total[u]);
#pragma unroll
              for (int i = 0; i < V; i++) acc[u][i] = fmaf(f, part[2 * R + r * DP + lane * V + i], acc[u][i]);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < TURNS; u++) {
          const uint32_t r = warp + u * NW;
          if (r >= rows) continue;
          const uint32_t tok = r / t.heads, head = t.head0 + r - tok * t.heads;
          float sum = total[u];
          if (p.a.sinks) sum += sink_weight(p.a.sinks, head, top[u]);
          const float unit = sum == 0.0f ? 0.0f : 1.0f / sum;
          T *out = (T *)p.out + (uint64_t)(t.row0 + t.token0 + tok) * p.out_stride + (uint64_t)head * D + lane * V;
#pragma unroll
          for (int i = 0; i < V; i += 2)
            if (lane * V + i < D) reinterpret_cast<uint32_t *>(out)[i / 2] = Num<T>::pack(acc[u][i] * unit, acc[u][i + 1] * unit);
        }
      }
    }
    // the rings are tiled copies' again
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (__syncthreads_or(join_lost)) break;
  }
  // The way out after a wait that has run out: nothing more is asked for, and what is in flight lands before the CTA ends.
  if (chunk_lost) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (lane < ST) drain_copies(&s_full[warp * ST + lane]);
  }
  if (join_lost) drain_copies(&s_join);
}

template <typename T, int DP>
cudaError_t launch_stream(const AttendParams &p, const PageMaps &maps, int sm_count, cudaStream_t s) {
  using S = StreamShape<DP>;
  constexpr size_t SMEM = 1024 + (size_t)16 * DP * 2 + (size_t)S::NW * S::ST * S::CHUNK;
  static_assert((size_t)S::NW * 16 * (DP + 10) * 4 <= (size_t)S::NW * S::ST * S::CHUNK, "the warps' results lie in the rings");
  const cudaError_t e = allow_smem<k_attend_stream<T, DP>>(SMEM);
  if (e != cudaSuccess) return e;
  return launch_overlapped(k_attend_stream<T, DP>, dim3(sm_count), S::THREADS, SMEM, s, false, p, maps);
}
template <typename T>
cudaError_t launch_stream(const AttendParams &p, const PageMaps &maps, int sm_count, cudaStream_t s) {
  if (p.a.head_dim <= 64) return launch_stream<T, 64>(p, maps, sm_count, s);
  return p.a.head_dim <= 128 ? launch_stream<T, 128>(p, maps, sm_count, s) : launch_stream<T, 256>(p, maps, sm_count, s);
}

}  // namespace

size_t attend_part_floats(int sm_count) {
  return std::max((size_t)2 * sm_count * part_floats(16, 256), attend_tc_part_floats(sm_count));
}
size_t attend_counts(int sm_count) { return (size_t)sm_count; }

cudaError_t launch_attend(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                          int sm_count, cudaStream_t s, int *launches) {
  // One row a sequence and no more heads of a key head than a tile has rows: the streaming kernel.  Any more rows: the tensor-core kernel, whose 128 rows a group cost
  // the same whatever they hold.
  if (kv.n_rows > kv.n_seqs || a.q_heads / a.kv_heads > 16) {
    *launches += 1;
    return launch_attend_tc(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
  }
  const PageMapShape m(a, kv, 16);
  PageMaps maps{};
  const bool mapped = encode_page_maps(&maps, m, a, kv);
  const AttendParams p{a, kv, q, out, q_stride, out_stride, ws, TileShape(a.q_heads, a.kv_heads, 16, START_UNITS, 1, 0, WHOLE_BLOCKS), mapped ? m.rows : 0, m.head_first};
  *launches += 1;
  return a.cache_type == MER_VALUE_F16 ? launch_stream<__half>(p, maps, sm_count, s) : launch_stream<__nv_bfloat16>(p, maps, sm_count, s);
}
