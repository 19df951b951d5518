// Attention of few new rows over a paged cache: single tokens, drafts.  Any head size up to 256 in steps of 8.
//
//   o = sum_j 2^(s_j - m) v_j / (sum_j 2^(s_j - m) [+ 2^(sink - m)]),  s_j = q . k_j * scale * log2 e,  m = max_j s_j
//
// in one pass over the keys with the running maximum and sum of every row.  What bounds it is reading the cache: per 16 tokens 16 * 2 *
// head_dim values for at most 32 rows of work.  So a warp is a stream of its own: it copies the next chunks of 16 tokens (tiled copies of 8 or 16
// tokens of a page; row by row, 16 bytes a lane, where a sequence's end or a window cuts a chunk or pages have no such runs) into a ring that no other warp sees, multiplies the one that has landed (mma.sync on 16 x 16 tiles; at this rate of
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

constexpr uint32_t START_UNITS = 2;  // what a tile costs beside its blocks, in blocks

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

// Rows of a tile are MT * 16, warps NW, chunks in flight per warp ST.
template <int DP>
struct StreamShape {
  static constexpr int NW = DP == 256 ? 4 : 8, ST = DP == 64 ? 6 : 3;
  static constexpr uint32_t KB = NW * 16, THREADS = NW * 32, CHUNK = 2 * 16 * DP * 2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// Byte offset of 16-byte piece `c` of row `r` of ROWS: 64 values of every row, then the next 64, in the 128-byte swizzle; eight rows of one
// column of pieces lie in eight different bank groups.
template <uint32_t ROWS>
__device__ __forceinline__ uint32_t piece(uint32_t r, uint32_t c) {
  return (c >> 3) * (ROWS * 128) + r * 128 + (((c ^ r) & 7) << 4);
}

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(StreamShape<DP>::THREADS, 1) k_attend_stream(const AttendParams p, const __grid_constant__ PageMaps maps) {
  using S = StreamShape<DP>;
  constexpr int NW = S::NW, ST = S::ST, R = MT * 16;
  constexpr uint32_t KB = S::KB, THREADS = S::THREADS;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ uint64_t s_full[NW * ST];  // a chunk has landed: every lane of its warp arrives
  __shared__ RunFound s_found;
  __shared__ uint32_t s_flag;
  uint8_t *s_ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);  // [NW][ST][k, v][DP / 64][16][64]
  uint8_t *s_q = s_ring + NW * ST * S::CHUNK;                                  // [DP / 64][R][64]
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t D = p.a.head_dim, page_tokens = p.a.page_tokens, window = p.a.window;
  const TileShape &ts = p.ts;
  for (uint32_t i = tid; i < NW * ST; i += THREADS) mbar_init(&s_full[i], 32);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  grid_dep_wait();
  grid_dep_launch();
  const RunStart run = find_run<KB, THREADS>(p.kv, ts, window, blockIdx.x, gridDim.x, 1, s_found);
  if (blockIdx.x == 0) clear_rows_without_place<T, THREADS>(p.a, p.kv, (T *)p.out, p.out_stride, p.ws.status);
  if (blockIdx.x >= run.parts) return;
  RunWalk<KB> walk(p.kv, ts, window, run);
  const float to_log2 = p.a.scale * LOG2E;
  uint32_t fill = 0, stage = 0, stage_phase = 0, timed_out = 0;  // of the warp's ring: what is asked for next, what is taken next
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
        cp_async16(dst + piece<16>(r, c), (const char *)p.kv.k_pages + off, in ? 16 : 0);
        cp_async16(dst + 16 * DP * 2 + piece<16>(r, c), (const char *)p.kv.v_pages + off, in ? 16 : 0);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    };
    uint32_t ahead[ST];
#pragma unroll
    for (int i = 0; i < ST; i++) ahead[i] = entry(t.lo + i);
#pragma unroll
    for (int i = 0; i < ST - 1; i++) issue(t.lo + i, ahead[i]);
    uint32_t next_entry = ahead[ST - 1];
    // ---- queries, while the first chunks are on their way
    for (uint32_t i = tid; i < R * (DP / 8); i += THREADS) {
      const uint32_t r = i / (DP / 8), c = i % (DP / 8), tok = r / t.heads, h = r - tok * t.heads;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows && c * 8 < D)
        v = __ldg(reinterpret_cast<const uint4 *>((const T *)p.q + (uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + h) * D + c * 8));
      *reinterpret_cast<uint4 *>(s_q + piece<R>(r, c)) = v;
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
    for (uint32_t blk = t.lo; blk < t.hi; blk++) {
      {
        const uint32_t number = next_entry;
        next_entry = entry(blk + ST);
        __syncwarp();  // the chunk that lay in this stage has been read
        issue(blk + ST - 1, number);
      }
      if (!wanted(blk)) continue;
      const uint32_t key0 = blk * KB + warp * 16, base = ring + stage * S::CHUNK;
      timed_out |= !mbar_wait(&s_full[warp * ST + stage], stage_phase);
      stage = stage + 1 == ST ? 0 : stage + 1, stage_phase ^= stage == 0;
      float s[MT][2][4];
      {
        // One tile of rows: the products of even and odd pieces of a head apart, so that half as many wait for one another.
        constexpr int CHAINS = MT == 1 ? 2 : 1;
        float c[CHAINS][MT][2][4];
#pragma unroll
        for (int i = 0; i < CHAINS * MT * 8; i++) (&c[0][0][0][0])[i] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) {
          uint32_t kf[4];
          ldm4(kf, base + piece<16>((lane / 16) * 8 + (lane & 7), kk * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int mt = 0; mt < MT; mt++) {
            uint32_t qf[4];
            ldm4(qf, q_addr + piece<R>(mt * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), kk * 2 + (lane >> 4)));
            mma16816<T>(c[kk % CHAINS][mt][0], qf, kf[0], kf[1]);
            mma16816<T>(c[kk % CHAINS][mt][1], qf, kf[2], kf[3]);
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[mt][n][e] = CHAINS == 2 ? c[0][mt][n][e] + c[CHAINS - 1][mt][n][e] : c[0][mt][n][e];
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
        ldm4_trans(vf, vbase + piece<16>(((lane >> 3) & 1) * 8 + (lane & 7), dn * 2 + (lane >> 4)));
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          mma16816<T>(o[mt][2 * dn], pf[mt], vf[0], vf[1]);
          mma16816<T>(o[mt][2 * dn + 1], pf[mt], vf[2], vf[3]);
        }
      }
    }
    if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
    // ---- the warps' results: [warp][row] maximum and sum, [warp][row][DP] output, where the rings were
    constexpr int OP = DP + 8;  // floats of a row of it: the rows of a fragment lie in different banks
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
        if (r >= rows) continue;
        if ((lane & 3) == 0) s_m[warp * R + r] = m[mt][e], s_l[warp * R + r] = sum;
#pragma unroll
        for (int i = 0; i < DP / 8; i++)
          *reinterpret_cast<float2 *>(s_o + ((size_t)warp * R + r) * OP + i * 8 + (lane & 3) * 2) = make_float2(o[mt][i][2 * e], o[mt][i][2 * e + 1]);
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
      // The CTA that arrives last joins the parts in the order of the runs and leaves the count at zero: a warp a row, its lanes first over the parts (their
      // factors), then over the row's values.
      uint32_t c0, n;
      runs_of_tile(run, t, &c0, &n);
      if (tid == 0) {
        const bool is_last = arrive_acq_rel(p.ws.counts + c0) + 1 == n;
        if (is_last) p.ws.counts[c0] = 0;
        s_flag = is_last;
      }
      __syncthreads();
      if (s_flag) {
        constexpr int V = DP / 32;  // values of a lane
        const float *first = part_of_tile(run, t, p.ws.parts, c0, 0, part_floats(R, DP)), *others = part_of_tile(run, t, p.ws.parts, c0, 1, part_floats(R, DP));
        auto part_of = [&](uint32_t k) { return k == 0 ? first : others + (size_t)(k - 1) * (2 * part_floats(R, DP)); };
        for (uint32_t r = warp; r < rows; r += NW) {
          // a lane's values of AT_ONCE parts are asked for before the parts' maxima are known
          constexpr uint32_t AT_ONCE = V == 8 || MT == 2 ? 8 : 16;
          float top = -INFINITY, total = 0.0f, acc[V], v[AT_ONCE][V];
          auto ask = [&](uint32_t k0) {
#pragma unroll
            for (uint32_t k = 0; k < AT_ONCE; k++) {
              if (k0 + k >= n) continue;
              const float *row = part_of(k0 + k) + 2 * R + (size_t)r * DP + lane * V;
              if constexpr (V == 2)
                *reinterpret_cast<float2 *>(v[k]) = __ldcg(reinterpret_cast<const float2 *>(row));
              else
#pragma unroll
                for (int i = 0; i < V; i += 4) *reinterpret_cast<float4 *>(v[k] + i) = __ldcg(reinterpret_cast<const float4 *>(row + i));
            }
          };
          ask(0);
          for (uint32_t k = lane; k < n; k += 32) top = fmaxf(top, __ldcg(part_of(k) + r));
#pragma unroll
          for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
#pragma unroll
          for (int i = 0; i < V; i++) acc[i] = 0.0f;
          float f = 0.0f;  // of part (k0 rounded down to 32) + lane
          for (uint32_t k0 = 0; k0 < n; k0 += AT_ONCE) {
            if (k0 % 32 == 0) {
              f = 0.0f;
              if (k0 + lane < n) {
                const float *from = part_of(k0 + lane);
                const float mk = __ldcg(from + r);
                f = mk == -INFINITY ? 0.0f : exp2_approx(mk - top);
                total = fmaf(f, __ldcg(from + R + r), total);
              }
            }
            if (k0) ask(k0);
#pragma unroll
            for (uint32_t k = 0; k < AT_ONCE; k++) {
              const float fk = __shfl_sync(0xFFFFFFFFu, f, (k0 + k) & 31);
#pragma unroll
              for (int i = 0; i < V; i++)
                if (k0 + k < n) acc[i] = fmaf(fk, v[k][i], acc[i]);
            }
          }
#pragma unroll
          for (int d = 16; d; d /= 2) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
          const uint32_t tok = r / t.heads, head = t.head0 + r - tok * t.heads;
          if (p.a.sinks) total += exp2_approx(__ldg(p.a.sinks + head) * LOG2E - top + P_SHIFT);
          const float unit = total == 0.0f ? 0.0f : 1.0f / total;
          T *out = (T *)p.out + (uint64_t)(t.row0 + t.token0 + tok) * p.out_stride + (uint64_t)head * D + lane * V;
#pragma unroll
          for (int i = 0; i < V; i += 2)
            if (lane * V + i < D) reinterpret_cast<uint32_t *>(out)[i / 2] = Num<T>::pack(acc[i] * unit, acc[i + 1] * unit);
        }
      }
    }
    // the rings are tiled copies' again
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
  if (timed_out) atomicOr(p.ws.status, MER_DEVSTAT_TIMEOUT);
}

template <typename T, int DP, int MT>
cudaError_t launch_stream(const AttendParams &p, const PageMaps &maps, int sm_count, cudaStream_t s) {
  using S = StreamShape<DP>;
  constexpr size_t SMEM = 1024 + (size_t)MT * 16 * DP * 2 + (size_t)S::NW * S::ST * S::CHUNK;
  static_assert((size_t)S::NW * MT * 16 * (DP + 10) * 4 <= (size_t)S::NW * S::ST * S::CHUNK, "the warps' results lie in the rings");
  const cudaError_t e = allow_smem<k_attend_stream<T, DP, MT>>(SMEM);
  if (e != cudaSuccess) return e;
  return launch_overlapped(k_attend_stream<T, DP, MT>, dim3(sm_count), S::THREADS, SMEM, s, false, p, maps);
}
template <typename T>
cudaError_t launch_stream(const AttendParams &p, const PageMaps &maps, int sm_count, cudaStream_t s) {
  if (p.a.head_dim <= 64) return launch_stream<T, 64, 1>(p, maps, sm_count, s);
  return p.a.head_dim <= 128 ? launch_stream<T, 128, 1>(p, maps, sm_count, s) : launch_stream<T, 256, 1>(p, maps, sm_count, s);
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
  if (a.head_dim <= 128 && (kv.n_rows > kv.n_seqs || a.q_heads / a.kv_heads > 16)) {
    *launches += 1;
    return launch_attend_tc(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
  }
  const PageMapShape m(a, kv, 16);
  PageMaps maps{};
  const bool mapped = encode_page_maps(&maps, m, a, kv);
  const AttendParams p{a, kv, q, out, q_stride, out_stride, ws, TileShape(a.q_heads, a.kv_heads, 16, START_UNITS, 1, 0), mapped ? m.rows : 0, m.head_first};
  *launches += 1;
  return a.cache_type == MER_VALUE_F16 ? launch_stream<__half>(p, maps, sm_count, s) : launch_stream<__nv_bfloat16>(p, maps, sm_count, s);
}
