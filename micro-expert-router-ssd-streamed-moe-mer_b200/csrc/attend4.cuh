// Attention of a few new tokens a sequence over a paged cache of 4 bits.  Head sizes up to 256 in steps of 8.
//
//   o = sum_j p_j v_j / (sum_j p_j [+ sink]),  p_j = 2^(s_j - m),  s_j = q . k_j * scale * log2 e,  m = max_j s_j
//
// in one pass, as in kernels_attend.cu: a warp is a stream of its own, chunks of 16 tokens, maximum, sum and output of its own tokens in registers.  Reading a token's
// codes takes a third of a 16-bit cache's time, so the instructions that unpack are what counts, and codes are multiplied as they are:
//
//   * A code's four bits, masked in place, are an f16 number: a subnormal one, code * 2^-24 or code * 2^-20 as they stand in the lower or the upper half of a byte, which the matrix
//     units multiply exactly.
//   * Keys:  q . k = sum_g scale_g (q . code)_g + minimum_g (sum of q)_g.  One AND makes two operands' values, and every second word a shift before that.  The first product is exact
//     in fp32 and takes its scale there; the second is one more matrix product, whose operand the words (scale, minimum) are as they lie in memory, against (0, sum of q) in two
//     parts of f16.
//   * Values:  o = sum_g (p scale_g) . code + p . minimum_g.  Operands are a code and that code with sixteen times the next one (a byte as it is: 2^-24 (code + 16 next)), which the
//     end takes apart again: four instructions a word, where the codes alone are five.  A weight times a scale is rounded to f16, the weights themselves once more; minima are an operand as above.
//     Minima and codes have opposite signs, so that the first of these roundings would count more than twice.  For f16 outputs what the products lose, sum p scale_g - sum f16(p scale_g), is
//     added up beside the minima (their operand has the scales, one more product takes the rounded ones away) and given back to the middle of the codes, 7.5 times: 64 tokens behind 800 to
//     8000 are off by 0.00036 of their norm, 0.00054 without it, for one matrix product a group and chunk (40 tokens of 64 and 4 heads of 80
//     35.3 us, 34.5 without).  bf16 outputs round to 0.0017 themselves.
//   * Both products have tokens or the head's values along M and the rows along N, so that eight rows cost half of sixteen; the weights are transposed between them (movmatrix).
//   * Queries are f16 divided by a power of two of their row.  A row's reference m follows its maximum only when that has grown by more than 2^LAG4.  Weights are made as
//     2^(s - m + 10): a weight is below 2^14, its product with a scale below 4 fits f16, and small ones lie above its last bit for 2^-34 of the largest.  Where a product did not fit
//     (an output that is not finite says so), the warp takes its blocks of the tile three times more, weights and reference as they were: each time the scales of one class, below 4, below
//     256 and the others, times 1, 2^-6 and 2^-12, all of which fit and none of which loses a bit.  (Weights 2^13 times smaller in one more pass lost those below 2^-22 of the largest:
//     the sum had them, the output did not.)  A product lies above f16's last bit for weights down to 2^-34 of the largest divided by its scale; what equal ones below that sum to is lost to
//     bf16 outputs, where values are as small as 1e-4 and thousands of tokens share the rest of a row.
//
// A warp's ring of chunks is seen by no other warp.  Where pages are whole chunks (multiples of 16 tokens) a lane makes a chunk's four bulk copies: the addresses of several chunks are
// one instruction stream, so that a chunk costs a dozen instructions for its copies instead of sixty (copies of 16 bytes by every lane: 54 us for 64 tokens behind 800 to 8000, 49
// so, before values' codes were multiplied by pairs).  Other pages: cp.async of 16 bytes a lane, token by token.
//
// 32 and 4 heads of 128 in bf16, groups of 32, pages of 16: captured: 64 tokens behind 800 to 8000 45.7 us = 3.3 TB/s (16 bits: 81.9 us), one behind 32000 22.5 us (18.4).  What bounds it: issuing.  A chunk is
// 335 instructions, half of them on the ALU (2.4 cycles each for a quarter of an SM; an mma 5.8), and takes 296 ns a quarter of an SM, whatever the number of warps: 5.1 TB/s if it went on
// all the time.  The rest is 6 us until the first chunk has landed, 2 us of switching for every tile that a CTA goes through, and CTAs that end before others.
#pragma once

#include <cuda_runtime.h>

#include <cfloat>
#include <type_traits>

#include "attend_join.cuh"
#include "attend_wait.cuh"
#include "attention.cuh"
#include "kernels.h"
#include "kv4_unpack.cuh"
#include "ptx.cuh"

namespace {

constexpr float LAG4 = 4.0f, SHIFT4 = 14.0f - LAG4;

struct Attend4Params {
  AttnLayer a;
  KvBatchDev kv;
  const void *q;
  void *out;
  uint64_t q_stride, out_stride;
  AttnWorkspace ws;
  TileShape ts;
  uint32_t min_units;
};

// U: units of 32 values, GS: 1 where two units share a scale, NT: eights of rows.
template <int U, int GS, int NT>
struct Stream4Shape {
  static constexpr bool SMALL = U <= 4 && NT == 1;  // 128 registers a thread do
  static constexpr int NW = SMALL ? 8 : 4, CTAS = 2;
  static constexpr int G = (U + GS) >> GS, R = 8 * NT, TILES = 2 * U;
  static constexpr uint32_t KB = NW * 16, THREADS = NW * 32;
  static constexpr uint32_t CODES = 16 * 16 * U, SCALES = 16 * 4 * G, CHUNK = 2 * (CODES + SCALES);  // keys' codes and scales, values' codes and scales
  static constexpr int ST = U == 2 && NT == 1 ? 8 : 4;
  static constexpr uint32_t RING = NW * ST * CHUNK, OP = 32 * U + 4;
  static constexpr uint32_t JOIN = NW * R * (OP + 2) * 4;  // the warps' maxima, sums and outputs
  static constexpr uint32_t MAX_PARTS = RING / 4 / R - 2;  // of a tile: their weights lie in the ring, and the rows' sums
  static constexpr size_t SMEM = RING > JOIN ? RING : JOIN;
  static constexpr size_t SM_FLOATS = (size_t)2 * CTAS * part_floats(R, 32 * U);  // of parts that an SM's CTAs may leave
};
constexpr size_t ATTEND4_SM_FLOATS = Stream4Shape<8, 0, 2>::SM_FLOATS;  // the most of all shapes

// The chunk's token that has place `slot` of eight among the products' rows: neighbours are one even and one odd token, whose codes lie in different banks.
__device__ __forceinline__ constexpr uint32_t token_of(uint32_t slot) { return slot ^ ((slot >> 1) & 1); }

template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(in ? N : 0) : "memory");
}
__device__ __forceinline__ void bulk_to(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void sts_zero(uint32_t a) { asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory"); }
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
// N 32-bit words from an address on a multiple of 4 N (at most 16) bytes.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = lds128(a + i * 4);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 v = lds64(a + i * 4);
      w[i] = v.x, w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = lds32(a + i * 4);
  }
}
// A scale and its minimum in a pass over one class of scales: what is below 4 (pass 1), below 256 times 2^-6 (2), the others times 2^-12 (3), and zero for what is in another class.
// Minima are the first class's.
__device__ __forceinline__ void scales_of_pass(uint32_t at, uint32_t pass) {
  const uint32_t word = lds32(at), size = word & 0x7FFFu, of = size < 0x4400u ? 1u : size < 0x5C00u ? 2u : 3u;
  const __half scale = __hmul(__ushort_as_half((uint16_t)word), __ushort_as_half(pass == 1 ? 0x3C00 : pass == 2 ? 0x2400 : 0x0C00));
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"((of == pass ? (uint32_t)__half_as_ushort(scale) : 0u) | (pass == 1 ? word & 0xFFFF0000u : 0u)) : "memory");
}
// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// A value that is computed where it stands: nothing that is made of it moves in front of a branch that is hardly ever taken.
__device__ __forceinline__ uint32_t here(uint32_t v) {
  asm volatile("" : "+r"(v));
  return v;
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t t;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// WHOLE: pages are whole chunks of 16 tokens.  F16: queries and outputs are f16, else bf16.
template <int U, int GS, int NT, bool WHOLE, bool F16>
__global__ void __launch_bounds__(Stream4Shape<U, GS, NT>::THREADS, Stream4Shape<U, GS, NT>::CTAS) k_attend4(const __grid_constant__ Attend4Params p) {
  using S = Stream4Shape<U, GS, NT>;
  constexpr int NW = S::NW, ST = S::ST, R = S::R, G = S::G;
  constexpr uint32_t KB = S::KB, THREADS = S::THREADS;
  extern __shared__ __align__(128) uint8_t smem[];  // [NW][ST] chunks
  __shared__ RunFound s_found;
  __shared__ RunStart s_run;
  __shared__ RunPlace s_walk;
  __shared__ TileWork s_tile;  // here, not in registers: the loop over a tile's blocks needs all of these for itself.  tokens == 0: there is none left
  __shared__ uint32_t s_flag;
  __shared__ uint64_t s_full[NW * ST];  // a chunk has landed
  __shared__ uint32_t s_pass[NW];
  __shared__ volatile uint32_t s_stop;  // a wait has run out
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, eighth = lane >> 2;
  const uint32_t D = p.a.head_dim, page_tokens = p.a.page_tokens, window = p.a.window;
  constexpr bool f16 = F16;
  const TileShape &ts = p.ts;
  if (WHOLE && tid < NW * ST) mbar_init(&s_full[tid], 1);
  if (tid == 0) s_stop = 0;
  if (WHOLE) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  grid_dep_wait();
  grid_dep_launch();
  {
    const RunStart run = find_run<KB, THREADS>(p.kv, ts, window, blockIdx.x, gridDim.x, p.min_units, s_found);
    if (tid == 0) s_run = run, s_walk = RunWalk<KB>(p.kv, ts, window, run);
  }
  __syncthreads();
  const RunStart &run = s_run;
  if (blockIdx.x == 0) {
    if (f16)
      clear_rows_without_place<__half, THREADS>(p.a, p.kv, (__half *)p.out, p.out_stride, p.ws.status);
    else
      clear_rows_without_place<__nv_bfloat16, THREADS>(p.a, p.kv, (__nv_bfloat16 *)p.out, p.out_stride, p.ws.status);
  }
  if (blockIdx.x >= run.parts) return;
  const uint32_t ring = smem_u32(smem) + warp * (ST * S::CHUNK);
  const float to_log2 = p.a.scale * LOG2E;
  uint32_t bad = 0;
  bool lost = false;   // the warp has given up the wait for a chunk
  uint32_t taken = 0;  // chunks of the warp's so far: chunk n lies in stage n % ST
  const uint32_t key_token = token_of(eighth), even_token = token_of(quad * 2), odd_token = token_of(quad * 2 + 1);
  const TileWork &t = s_tile;
  for (;;) {
    if (tid == 0) {
      RunWalk<KB> walk(p.kv, ts, window, s_walk);
      TileWork next;
      if (!walk.next(&next)) next.tokens = 0;
      s_tile = next, s_walk = walk;
    }
    __syncthreads();
    if (t.tokens == 0) break;
    const uint32_t tile_rows = t.tokens * t.heads;
    const uint32_t end = t.past + t.token0 + t.tokens;  // behind the last token that a row of the tile sees
    const uint32_t start = first_seen(t, window);
    // ---- the warp's blocks are b_lo .. b_hi, a chunk each
    const uint32_t w16 = warp * 16;
    const uint32_t b_lo = max(t.lo, start < w16 + 16 ? 0u : (start - w16 - 16) / KB + 1), b_hi = end <= w16 ? t.lo : min(t.hi, (end - w16 + KB - 1) / KB);
    const uint32_t *const table = p.kv.page_table + (uint64_t)t.seq * p.kv.table_stride;
    // Queries are asked for ahead of the copies: behind these they would wait for a full ring of every SM.  Lane (eighth, quad) has values 32 u + 8 quad .. of row x * 8 + eighth.
    uint4 raw[NT][U];
#pragma unroll
    for (int x = 0; x < NT; x++) {
      const uint32_t r = x * 8 + eighth, tok = r / t.heads, h = r - tok * t.heads;
      const uint16_t *const row = (const uint16_t *)p.q + (uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + h) * D + quad * 8;
#pragma unroll
      for (int u = 0; u < U; u++) raw[x][u] = r < tile_rows && u * 32 + quad * 8 < D ? *reinterpret_cast<const uint4 *>(row + u * 32) : make_uint4(0, 0, 0, 0);
    }
    struct Place {
      uint32_t number, in;  // a page, and the token in it
    };
    // Where block `blk` is (WHOLE: its first token), or the lane's token of it.
    auto entry = [&](uint32_t blk) {
      const uint32_t key = blk * KB + w16 + (WHOLE ? 0 : lane & 15), slot = divided(key, p.kv.page_tokens);
      Place at;
      at.in = key - slot * page_tokens;
      at.number = blk < b_hi && (WHOLE || (key >= first_seen(t, window) && key < t.past + t.token0 + t.tokens)) && slot < p.kv.table_stride ? table[slot] : 0xFFFFFFFFu;
      return at;
    };
    const uint64_t head_at = t.kv_head * p.kv.head_stride;
    // WHOLE: lanes 0 .. count - 1 have a block each from `blk` on, chunk n of the warp's and the next ones.  Else all lanes have block `blk`.
    auto issue = [&](uint32_t blk, const Place &at, uint32_t n, uint32_t count) {
      if constexpr (WHOLE) {
        if (lane < count && blk + lane < b_hi) {
          const uint32_t stage = (n + lane) % ST, dst = ring + stage * S::CHUNK;
          uint64_t *const bar = &s_full[warp * ST + stage];
          if (at.number < p.kv.n_pages) {
            const uint64_t page = at.number * p.kv.page_stride + head_at, codes = page + at.in * (16 * U), scales = page + p.a.kv4.codes + at.in * (4 * G);
            const char *const k = (const char *)p.kv.k_pages, *const v = (const char *)p.kv.v_pages;
            mbar_expect_tx(bar, S::CHUNK);
            bulk_to(dst, k + codes, S::CODES, bar);
            bulk_to(dst + S::CODES, k + scales, S::SCALES, bar);
            bulk_to(dst + S::CODES + S::SCALES, v + codes, S::CODES, bar);
            bulk_to(dst + 2 * S::CODES + S::SCALES, v + scales, S::SCALES, bar);
          } else {  // no such page: scales and minima of zero
            bad = 1;
            for (uint32_t i = 0; i < S::SCALES; i += 16) sts_zero(dst + S::CODES + i), sts_zero(dst + 2 * S::CODES + S::SCALES + i);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // later copies go where these zeros are
            mbar_arrive(bar);
          }
        }
      } else {
        if (blk < b_hi) {
          constexpr int N = G % 4 == 0 ? 16 : G % 2 == 0 ? 8 : 4;
          const uint32_t end = t.past + t.token0 + t.tokens, start = first_seen(t, window), dst = ring + n % ST * S::CHUNK;
          const uint32_t key = blk * KB + w16 + (lane & 15);
          const bool seen = key >= start && key < end, there = seen && at.number < p.kv.n_pages;
          if (seen && !there) bad = 1;
          const uint64_t block = there ? at.number * p.kv.page_stride + head_at : 0;
          const uint32_t valid = __ballot_sync(0xFFFFFFFFu, there);  // tokens of the chunk, twice
#pragma unroll
          for (int i = 0; i < (U + 1) / 2; i++) {
            const uint32_t e = i * 32 + lane, tok = e / U % 16, c = e % U, to = tok * (16 * U) + c * 16;
            const uint64_t off = __shfl_sync(0xFFFFFFFFu, block, tok) + (uint64_t)__shfl_sync(0xFFFFFFFFu, at.in, tok) * (16 * U) + c * 16;
            if (U % 2 && e >= 16 * U) continue;
            const bool ok = valid >> tok & 1;
            copy16(dst + to, (const char *)p.kv.k_pages + (ok ? off : 0), ok ? 16 : 0);
            copy16(dst + S::CODES + S::SCALES + to, (const char *)p.kv.v_pages + (ok ? off : 0), ok ? 16 : 0);
          }
          // scales: lanes 0 .. 15 the keys', the others the values'
          const char *const src = (const char *)(lane < 16 ? p.kv.k_pages : p.kv.v_pages) + (there ? block + p.a.kv4.codes + (uint64_t)at.in * (4 * G) : 0);
          const uint32_t to = dst + S::CODES + (lane < 16 ? 0 : S::CODES + S::SCALES) + (lane & 15) * (4 * G);
#pragma unroll
          for (int i = 0; i < 4 * G / N; i++) {
            if constexpr (N == 16)
              copy16(to + i * N, src + (there ? i * N : 0), there ? 16 : 0);
            else
              cp_async_small<N>(to + i * N, src + (there ? i * N : 0), there);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    };
    Place next_place;
    // The first chunks of the ring.
    auto start_ring = [&] {
      if constexpr (WHOLE) {
        const Place at = entry(b_lo + lane);
        next_place = entry(b_lo + ST + lane);
        issue(b_lo, at, taken, ST);
      } else {
        Place ahead[ST];
#pragma unroll
        for (int i = 0; i < ST; i++) ahead[i] = entry(b_lo + i);
#pragma unroll
        for (int i = 0; i < ST - 1; i++) issue(b_lo + i, ahead[i], taken + i, 1);
        next_place = ahead[ST - 1];
      }
    };
    start_ring();
    // ---- queries as the product's B operand wants them: pair p of a lane's eight meets the codes from bits 4 p and 16 + 4 p on, which stand for themselves times 2^-24 where p is
    // even, 2^-20 where it is odd.
    uint32_t qf[NT][U][4], qs[NT][(G + 3) / 4][2];  // qs: sums of a group's queries in two parts, each behind a zero
    float row_factor[NT];  // of row x * 8 + eighth
#pragma unroll
    for (int x = 0; x < NT; x++) {
      auto pair = [&](uint32_t w) { return f16 ? __half22float2(as_half2(w)) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); };
      uint32_t words[U][4], most = 0;
#pragma unroll
      for (int u = 0; u < U; u++) {
        words[u][0] = raw[x][u].x, words[u][1] = raw[x][u].y, words[u][2] = raw[x][u].z, words[u][3] = raw[x][u].w;
#pragma unroll
        for (int e = 0; e < 4; e++) most = __vmaxu2(most, words[u][e] & 0x7FFF7FFFu);  // magnitudes have the order of their bits
      }
      float2 top2 = pair(most);
      float top = fmaxf(top2.x, top2.y);
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const uint32_t power = min(max(__float_as_uint(top) >> 23, 1u), 253u);
      const float per = __uint_as_float((254 - power) << 23);
      row_factor[x] = fmaxf(to_log2 * __uint_as_float(power << 23), FLT_MIN);  // a hidden score times it is one still
      float sums[G];
#pragma unroll
      for (int g = 0; g < G; g++) sums[g] = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 v = pair(words[u][e]);
          const __half2 n = __floats2half2_rn(v.x * per, v.y * per);
          sums[u >> GS] += __low2float(n) + __high2float(n);
          qf[x][u][e] = as_u32(e % 2 ? n : __hmul2(n, as_half2(0x4C004C00u)));  // 16
        }
#pragma unroll
      for (int g = 0; g < G; g++) {
        sums[g] += __shfl_xor_sync(0xFFFFFFFFu, sums[g], 1);
        sums[g] += __shfl_xor_sync(0xFFFFFFFFu, sums[g], 2);
      }
#pragma unroll
      for (int b = 0; b < (G + 3) / 4; b++) {
        float mine = 0.0f;
#pragma unroll
        for (int g = b * 4; g < G && g < b * 4 + 4; g++) mine = quad == g - b * 4 ? sums[g] : mine;
        const __half hi = __float2half_rn(mine);
        qs[x][b][0] = (uint32_t)__half_as_ushort(hi) << 16;
        qs[x][b][1] = (uint32_t)__half_as_ushort(__float2half_rn(mine - __half2float(hi))) << 16;
      }
    }
    // Every row sees the tokens all_from .. all_see; of the warp's chunks, those of blocks n_lo .. n_lo + n_all have no others.
    const uint32_t all_see = t.past + t.token0, all_from = window && end > window ? end - window : 0;
    const uint32_t n_lo = all_from <= w16 ? 0u : (all_from - w16 + KB - 1) / KB, n_hi = all_see < w16 + 15 ? 0u : (all_see - w16 - 15) / KB + 1, n_all = n_hi > n_lo ? n_hi - n_lo : 0;
    // The lane has rows x * 8 + quad * 2 + e of scores and outputs.  least: sums of weights times minima
    // A weight is 2^(s * factor - less) with less = m - SHIFT4; limit: the score from which on m has to follow, -infinity while there is no m.
    float o[NT][S::TILES][4], least[NT][4], less[NT][2], limit[NT][2], l[NT][2], factor[NT][2];
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
      for (int e = 0; e < 2; e++) factor[x][e] = __shfl_sync(0xFFFFFFFFu, row_factor[x], quad * 8 + e * 4);
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
      for (int e = 0; e < 2; e++) less[x][e] = 0.0f, limit[x][e] = -INFINITY;
    // s_pass 1 to 3: over one class of scales.  The references are the first pass's last ones and stay: no score is above what they allow.  What such a pass has beside the first one lies in
    // memory and behind the branch of blocks that need a mask, so that the loop has the registers it had (sums kept in registers: 64 tokens behind 800 to 8000 48.1 us, 45.7 so).
    if (lane == 0) s_pass[warp] = 0;
    float kept[NT * (S::TILES + 1) * 4];  // the passes' sums
    uint32_t n_n = n_all;
  again:
#pragma unroll
    for (int x = 0; x < NT; x++) {
#pragma unroll
      for (int e = 0; e < 2; e++) l[x][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; e++) least[x][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < S::TILES; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[x][i][e] = 0.0f;
    }
    for (uint32_t blk = b_lo; blk < b_hi; blk++) {
      if constexpr (WHOLE) {
        // the places of the two chunks in front are asked for again
        if (((blk - b_lo) & 1) == 0 && blk != b_lo) {
          __syncwarp();
          issue(blk + ST - 2, next_place, taken + ST - 2, 2);
          next_place = entry(blk + ST + lane);
        }
        uint64_t *const bar = &s_full[warp * ST + taken % ST];
        const uint32_t parity = taken / ST & 1;
        if (!__all_sync(0xFFFFFFFFu, mbar_try(smem_u32(bar), parity)) && !wait_or_stop(bar, parity, &s_stop, p.ws.status)) {
          lost = true;
          break;
        }
      } else {
        const Place at = next_place;
        next_place = entry(blk + ST);
        __syncwarp();  // the chunk that lay in this stage has been read
        issue(blk + ST - 1, at, taken + ST - 1, 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        __syncwarp();
      }
      const uint32_t base = ring + taken % ST * S::CHUNK;
      taken++;
      // ---- scores: s[x][T][e] of row x * 8 + quad * 2 + e and token T * 8 + key_token
      const uint32_t kscales = base + S::CODES, values = base + S::CODES + S::SCALES, vscales = values + S::CODES;
      float s[NT][2][2];
      {
        uint32_t words[2][U], sc[2][G];
#pragma unroll
        for (int T = 0; T < 2; T++) {
          lds_words<U>(base + (T * 8 + key_token) * (16 * U) + quad * (4 * U), words[T]);
          lds_words<G>(kscales + (T * 8 + key_token) * (4 * G), sc[T]);
        }
        float mins[NT][4];
#pragma unroll
        for (int b = 0; b < (G + 3) / 4; b++) {
          uint32_t w[2];
#pragma unroll
          for (int T = 0; T < 2; T++) w[T] = b * 4 + quad < G ? lds32(kscales + (T * 8 + key_token) * (4 * G) + (b * 4 + quad) * 4) : 0u;
#pragma unroll
          for (int x = 0; x < NT; x++) {
            if (b == 0)
              mma_f16_first(mins[x], w[0], w[1], w[0], w[1], qs[x][b][0], qs[x][b][1]);
            else
              mma_f16(mins[x], w[0], w[1], w[0], w[1], qs[x][b][0], qs[x][b][1]);
          }
        }
        float part[NT][4];
#pragma unroll
        for (int g = 0; g < G; g++) {
          float c[NT][4];
#pragma unroll
          for (int u = g << GS; u < ((g + 1) << GS) && u < U; u++) {
            const uint32_t w0 = words[0][u], w1 = words[1][u], v0 = w0 >> 8, v1 = w1 >> 8;
#pragma unroll
            for (int x = 0; x < NT; x++) {
              if (u == g << GS)
                mma_f16_first(c[x], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[x][u][0], qf[x][u][1]);
              else
                mma_f16(c[x], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[x][u][0], qf[x][u][1]);
              mma_f16(c[x], v0 & 0x000F000Fu, v1 & 0x000F000Fu, v0 & 0x00F000F0u, v1 & 0x00F000F0u, qf[x][u][2], qf[x][u][3]);
            }
          }
          const float s0 = __low2float(as_half2(sc[0][g])), s1 = __low2float(as_half2(sc[1][g]));
#pragma unroll
          for (int x = 0; x < NT; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[x][e] = g == 0 ? c[x][e] * (e < 2 ? s0 : s1) : fmaf(c[x][e], e < 2 ? s0 : s1, part[x][e]);
        }
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[x][e / 2][e % 2] = fmaf(part[x][e], 1048576.0f, mins[x][e]);
      }
      if (blk - n_lo >= n_n) {  // in the passes over classes of scales all blocks
        const uint32_t at = here(blk) * KB + w16 + key_token;
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t last = t.past + t.token0 + min(x * 8 + quad * 2 + e, t.tokens * t.heads - 1) / t.heads;  // that the row sees
#pragma unroll
            for (int T = 0; T < 2; T++)
              if (!(at + T * 8 <= last && (window == 0 || at + T * 8 + window > last))) s[x][T][e] = -INFINITY;
          }
        if constexpr (WHOLE) {  // what no row sees may be anything: its minima must not meet weights of zero
          const uint32_t key = here(blk) * KB + w16 + (lane & 15);
          if (lane < 16 && (key < first_seen(t, window) || key >= t.past + t.token0 + t.tokens))
            for (uint32_t i = 0; i < 4 * G; i += 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(vscales + lane * (4 * G) + i), "r"(0u) : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // later copies go where these zeros are
          __syncwarp();
        }
        if (const uint32_t pass = s_pass[warp]) {
#pragma unroll 1
          for (uint32_t i = here(lane); i < 16 * G; i += 32) scales_of_pass(vscales + i * 4, pass);
          if constexpr (WHOLE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
      }
      // ---- values' scales of the lane's tokens, by pairs, and the minima as an operand: row 2 g + 1 of it (row g where a token's words are no whole 16 bytes) has group g's
      uint32_t vs[2][G], least_of[4] = {0, 0, 0, 0};
      if constexpr (G % 4 == 0) {
        const uint32_t at = vscales + (token_of(lane & 7) + (lane & 8)) * (4 * G) + (G == 8 ? (lane >> 4) * 16 : 0);
        if constexpr (G == 8)
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(least_of[0]), "=r"(least_of[2]), "=r"(least_of[1]), "=r"(least_of[3]) : "r"(at) : "memory");
        else
          asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(least_of[0]), "=r"(least_of[2]) : "r"(at) : "memory");
        // its row 2 g has the scales of group g, and a lane those of its tokens
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
          for (int g = 0; g < G; g++) vs[T][g] = __shfl_sync(0xFFFFFFFFu, least_of[2 * T + g / 4], g % 4 * 8 + quad);
      } else {
#pragma unroll
        for (int T = 0; T < 2; T++) {
          uint32_t sc[2][G];
          lds_words<G>(vscales + (T * 8 + even_token) * (4 * G), sc[0]);
          lds_words<G>(vscales + (T * 8 + odd_token) * (4 * G), sc[1]);
#pragma unroll
          for (int g = 0; g < G; g++) vs[T][g] = __byte_perm(sc[0][g], sc[1][g], 0x5410);
          const uint32_t even = vscales + (T * 8 + even_token) * (4 * G) + (eighth % G) * 4, odd = vscales + (T * 8 + odd_token) * (4 * G) + (eighth % G) * 4;
          const uint32_t e = lds32(even), o = lds32(odd);
          least_of[2 * T] = __byte_perm(e, o, 0x7632);
          if (f16) least_of[2 * T + 1] = __byte_perm(e, o, 0x5410);
        }
      }
      // ---- weights
      bool grows = false;
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int e = 0; e < 2; e++) grows |= fmaxf(s[x][0][e], s[x][1][e]) > limit[x][e];
      if (__any_sync(0xFFFFFFFFu, grows)) {
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float top = fmaxf(s[x][0][e], s[x][1][e]);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            top *= factor[x][e];
            const bool first = limit[x][e] == -INFINITY;
            const float m = less[x][e] + SHIFT4, now = first ? top : fmaxf(top, m), f = first ? 0.0f : exp2_approx(m - now);
            less[x][e] = now == -INFINITY ? 0.0f : now - SHIFT4;
            limit[x][e] = now == -INFINITY ? now : (now + LAG4) / factor[x][e];
            l[x][e] *= f;
#pragma unroll
            for (int i = 0; i < S::TILES; i++) o[x][i][e] *= f, o[x][i][2 + e] *= f;
            least[x][e] *= f, least[x][2 + e] *= f;
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int x = 0; x < NT; x++) {
        float w[2][2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
          for (int T = 0; T < 2; T++) w[T][e] = exp2_approx(fmaf(s[x][T][e], factor[x][e], -less[x][e]));
          l[x][e] += w[0][e] + w[1][e];
        }
#pragma unroll
        for (int T = 0; T < 2; T++) pf[x][T] = transposed(Num<__half>::pack(w[T][0], w[T][1]));
      }
#pragma unroll
      for (int x = 0; x < NT; x++) mma_f16(least[x], least_of[0], least_of[1], least_of[2], least_of[3], pf[x][0], pf[x][1]);
      // ---- values: a lane has words eighth * U .. of its four tokens
      {
        uint32_t w[2][U];  // word u of the lane's two tokens, of 16 bits each
#pragma unroll
        for (int T = 0; T < 2; T++) {
          const uint32_t even = values + (T * 8 + even_token) * (16 * U) + eighth * (2 * U), odd = values + (T * 8 + odd_token) * (16 * U) + eighth * (2 * U);
          if constexpr (U == 3) {
#pragma unroll
            for (int u = 0; u < U; u++) w[T][u] = lds16(even + u * 2) | lds16(odd + u * 2) << 16;
          } else {
            uint32_t h[2][U / 2];
            lds_words<U / 2>(even, h[0]);
            lds_words<U / 2>(odd, h[1]);
#pragma unroll
            for (int u = 0; u < U; u++) w[T][u] = __byte_perm(h[0][u / 2], h[1][u / 2], u % 2 ? 0x7632 : 0x5410);
          }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
          // rows of a tile: a code, and that code with sixteen times the next one, which the end takes apart again: four instructions a word where the codes alone are five
          const uint32_t l0 = w[0][u] & 0x00FF00FFu, l1 = w[1][u] & 0x00FF00FFu, h0 = __byte_perm(w[0][u], 0, 0x4341), h1 = __byte_perm(w[1][u], 0, 0x4341);
#pragma unroll
          for (int x = 0; x < NT; x++) {
            const uint32_t b0 = as_u32(__hmul2(as_half2(pf[x][0]), as_half2(vs[0][u >> GS]))), b1 = as_u32(__hmul2(as_half2(pf[x][1]), as_half2(vs[1][u >> GS])));
            mma_f16(o[x][2 * u], l0 & 0x000F000Fu, l0, l1 & 0x000F000Fu, l1, b0, b1);
            mma_f16(o[x][2 * u + 1], h0 & 0x000F000Fu, h0, h1 & 0x000F000Fu, h1, b0, b1);
            if (f16 && u % (1 << GS) == 0) {  // what the weights times scales have lost
              const int g = u >> GS;
              const uint32_t minus = eighth == (G % 4 == 0 ? g % 4 * 2 : g) ? 0xBC00BC00u : 0u;  // -1
              if (G % 4 == 0 && g < 4)
                mma_f16(least[x], minus, 0u, minus, 0u, b0, b1);
              else
                mma_f16(least[x], 0u, minus, 0u, minus, b0, b1);
            }
          }
        }
      }
    }
    if constexpr (!WHOLE) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if (!lost) {
      const uint32_t pass = s_pass[warp];
      bool odd = pass == 1 || pass == 2;
      if (pass == 0) {
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int i = 0; i < S::TILES; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) odd |= !(fabsf(o[x][i][e]) <= FLT_MAX);
      } else {
        asm volatile("" ::"l"(kept) : "memory");
        const float unit = pass == 1 ? 1.0f : pass == 2 ? 0x1p6f : 0x1p12f;
        auto keep = [&](float &v, int i) { kept[i] = v = pass == 1 ? v : fmaf(v, unit, kept[i]); };
#pragma unroll
        for (int x = 0; x < NT; x++) {
#pragma unroll
          for (int i = 0; i < S::TILES; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) keep(o[x][i][e], (x * (S::TILES + 1) + i) * 4 + e);
#pragma unroll
          for (int e = 0; e < 4; e++) keep(least[x][e], (x * (S::TILES + 1) + S::TILES) * 4 + e);
        }
        asm volatile("" ::"l"(kept) : "memory");
      }
      if (__any_sync(0xFFFFFFFFu, odd)) {  // a weight times a scale that f16 has no room for, or scores that are no numbers
        n_n = 0;
        __syncwarp();
        if (lane == 0) s_pass[warp] = pass + 1;
        __syncwarp();
        start_ring();
        goto again;
      }
    }
    // ---- the warps' results: [warp][row] reference and sum, [warp][row][OP] output, where the rings were
    if (__syncthreads_or(lost)) break;  // copies may still land in the rings
    const uint32_t rows = t.tokens * t.heads;
    float *const s_m = reinterpret_cast<float *>(smem), *const s_l = s_m + NW * R, *const s_o = s_l + NW * R;
#pragma unroll
    for (int x = 0; x < NT; x++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float sum = l[x][e];
#pragma unroll
        for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        const uint32_t r = x * 8 + quad * 2 + e;
        if (eighth == 0 && r < rows) s_m[warp * R + r] = limit[x][e] == -INFINITY ? limit[x][e] : less[x][e] + P_SHIFT, s_l[warp * R + r] = sum;  // the reference that the joins count with
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int g = u >> GS, at = G % 4 == 0 && g >= 4 ? 2 : 0, src = G % 4 == 0 ? (g % 4 * 2 + 1) * 4 : g * 4;
        float l0 = __shfl_sync(0xFFFFFFFFu, least[x][at], src + quad), l1 = __shfl_sync(0xFFFFFFFFu, least[x][at + 1], src + quad);
        if (f16) {
          const int lost_at = G % 4 == 0 ? at : 2, lost_src = G % 4 == 0 ? src - 4 : src;
          l0 = fmaf(7.5f, __shfl_sync(0xFFFFFFFFu, least[x][lost_at], lost_src + quad), l0), l1 = fmaf(7.5f, __shfl_sync(0xFFFFFFFFu, least[x][lost_at + 1], lost_src + quad), l1);
        }
        constexpr float CODE = 16777216.0f, NEXT = 1048576.0f;  // 2^24, and 2^20: sixteen times the code
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t row = x * 8 + quad * 2 + e;
          const float of_group = e ? l1 : l0;
          if (row < rows)
            *reinterpret_cast<float4 *>(s_o + ((size_t)warp * R + row) * S::OP + u * 32 + eighth * 4) =
                make_float4(fmaf(o[x][2 * u][e], CODE, of_group), fmaf(o[x][2 * u][2 + e] - o[x][2 * u][e], NEXT, of_group), fmaf(o[x][2 * u + 1][e], CODE, of_group),
                            fmaf(o[x][2 * u + 1][2 + e] - o[x][2 * u + 1][e], NEXT, of_group));
        }
      }
    }
    __syncthreads();
    const bool whole = t.lo == t.tile_lo && t.hi == t.tile_hi;
    constexpr int DP = 32 * U;
    float *part = p.ws.parts + (size_t)part_slot(run, t, blockIdx.x) * part_floats(R, DP);
    for (uint32_t i = tid; i < rows * (DP / 4); i += THREADS) {
      const uint32_t r = i / (DP / 4), c = i % (DP / 4) * 4;
      float reference = -INFINITY, sum = 0.0f;
      float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < NW; w++) reference = fmaxf(reference, s_m[w * R + r]);
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float mw = s_m[w * R + r], f = mw == -INFINITY ? 0.0f : exp2_approx(mw - reference);
        const float4 v = *reinterpret_cast<const float4 *>(s_o + ((size_t)w * R + r) * S::OP + c);
        sum = fmaf(f, s_l[w * R + r], sum);
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
      }
      if (whole) {
        if (f16)
          store_row<__half>(p.a, t, r, c, reference, sum, acc, (__half *)p.out, p.out_stride);
        else
          store_row<__nv_bfloat16>(p.a, t, r, c, reference, sum, acc, (__nv_bfloat16 *)p.out, p.out_stride);
      } else {
        if (c == 0) part[r] = reference, part[R + r] = sum;
        *reinterpret_cast<float4 *>(part + 2 * R + (size_t)r * DP + c) = acc;
      }
    }
    if (!whole) {
      __syncthreads();
      // The CTA that arrives last joins the parts in the order of the runs and leaves the count at zero.
      uint32_t c0, n;
      runs_of_tile(run, t, &c0, &n);
      if (tid == 0) {
        const bool is_last = arrive_acq_rel(p.ws.counts + c0) + 1 == n;
        if (is_last) p.ws.counts[c0] = 0;
        s_flag = is_last;
      }
      __syncthreads();
      if (s_flag) {
        // The parts' weights and the rows' sums first, a warp a row, then the outputs, every thread four values of a row: PARTS loads of it in flight.
        constexpr uint32_t PARTS = 8;
        float *const s_weight = reinterpret_cast<float *>(smem), *const s_sum = s_weight + R * n;  // [R][n], [R]
        const uint32_t floats = part_floats(R, DP);
        for (uint32_t r = warp; r < rows; r += NW) {
          float reference = -INFINITY, sum = 0.0f;
          for (uint32_t k = lane; k < n; k += 32) {
            const float m = __ldcg(part_of_tile(run, t, p.ws.parts, c0, k, floats) + r);
            s_weight[r * n + k] = m, reference = fmaxf(reference, m);
          }
#pragma unroll
          for (int d = 16; d; d /= 2) reference = fmaxf(reference, __shfl_xor_sync(0xFFFFFFFFu, reference, d));
          for (uint32_t k = lane; k < n; k += 32) {
            const float m = s_weight[r * n + k], f = m == -INFINITY ? 0.0f : exp2_approx(m - reference);
            s_weight[r * n + k] = f, sum = fmaf(f, __ldcg(part_of_tile(run, t, p.ws.parts, c0, k, floats) + R + r), sum);
          }
#pragma unroll
          for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
          if (lane == 0) s_sum[r] = sum, s_sum[R + r] = reference;
        }
        __syncthreads();
        for (uint32_t i = tid; i < rows * (DP / 4); i += THREADS) {
          const uint32_t r = i / (DP / 4), c = i % (DP / 4) * 4;
          float4 acc = make_float4(0, 0, 0, 0);
          for (uint32_t k0 = 0; k0 < n; k0 += PARTS) {
            float4 v[PARTS];
#pragma unroll
            for (uint32_t k = 0; k < PARTS; k++)
              v[k] = k0 + k < n ? __ldcg(reinterpret_cast<const float4 *>(part_of_tile(run, t, p.ws.parts, c0, k0 + k, floats) + 2 * R + (size_t)r * DP + c)) : make_float4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t k = 0; k < PARTS; k++) {
              const float f = k0 + k < n ? s_weight[r * n + k0 + k] : 0.0f;
              acc.x = fmaf(f, v[k].x, acc.x), acc.y = fmaf(f, v[k].y, acc.y), acc.z = fmaf(f, v[k].z, acc.z), acc.w = fmaf(f, v[k].w, acc.w);
            }
          }
          if (f16)
            store_row<__half>(p.a, t, r, c, s_sum[R + r], s_sum[r], acc, (__half *)p.out, p.out_stride);
          else
            store_row<__nv_bfloat16>(p.a, t, r, c, s_sum[R + r], s_sum[r], acc, (__nv_bfloat16 *)p.out, p.out_stride);
        }
      }
    }
    if constexpr (WHOLE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();  // the rings are copied into again
  }
  if (lost && lane < ST) drain_copies(&s_full[warp * ST + lane]);
  if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
}

template <int U, int GS, int NT>
cudaError_t launch_stream4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws, int sm_count, cudaStream_t s) {
  using S = Stream4Shape<U, GS, NT>;
  static_assert(S::CTAS <= ATTEND_CTAS && S::SM_FLOATS <= ATTEND4_SM_FLOATS, "the workspace has room for every CTA's count and parts");
  const Attend4Params p{a, kv, q, out, q_stride, out_stride, ws, TileShape(a.q_heads, a.kv_heads, S::R, ATTEND4_START, 1, 0, ATTEND4_WHOLE), ATTEND4_MIN_RUN};
  const auto launch = [&](auto whole, auto f16) {
    constexpr bool WHOLE = decltype(whole)::value, F16 = decltype(f16)::value;
    const cudaError_t e = allow_smem<k_attend4<U, GS, NT, WHOLE, F16>>(S::SMEM);
    return e != cudaSuccess ? e : launch_overlapped(k_attend4<U, GS, NT, WHOLE, F16>, dim3(std::min((uint32_t)(sm_count * S::CTAS), S::MAX_PARTS)), S::THREADS, S::SMEM, s, false, p);
  };
  if (a.cache_type == MER_VALUE_F16) return a.page_tokens % 16 == 0 ? launch(std::true_type{}, std::true_type{}) : launch(std::false_type{}, std::true_type{});
  return a.page_tokens % 16 == 0 ? launch(std::true_type{}, std::false_type{}) : launch(std::false_type{}, std::false_type{});
}

}  // namespace
