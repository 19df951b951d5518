// Attention of single new tokens over a paged cache of 4 bits.  Head sizes up to 256 in steps of 8.
//
//   o = sum_j p_j v_j / (sum_j p_j [+ sink]),  p_j = 2^(s_j - m),  s_j = q . k_j * scale * log2 e,  m = max_j s_j
//
// in one pass, as in kernels_attend.cu: a warp is a stream of its own, chunks of 16 tokens, maximum, sum and output of its own tokens in registers.  Reading a token's
// codes takes a quarter of a 16-bit cache's time, so the instructions that unpack are what counts, and codes are multiplied as they are:
//
//   * A code's four bits, masked in place, are an f16 number: a subnormal one, code * 2^-24 or code * 2^-20 as they stand in the lower or the upper half of a byte, which the matrix
//     units multiply exactly.  One AND makes two operands' values, and every second word a shift before that.
//   * Keys:  q . k = sum_g scale_g (q . code)_g + minimum_g (sum of q)_g.  The first product is exact in fp32 and takes its scale there; the second is one more
//     matrix product, whose operand the words (scale, minimum) are as they lie in memory, against (0, sum of q) in two parts of f16.
//   * Values:  o = sum_g (p scale_g) . code + p . minimum_g.  A weight times a scale is rounded to f16, the weights themselves once more; minima are an operand as above.
//   * Both products have tokens or the head's values along M and the rows along N, so that eight rows cost half of sixteen; the weights are transposed between them (movmatrix).
//   * Queries are f16 divided by a power of two of their row.  A row's reference m follows its maximum only when that has grown by more than 2^LAG4.  Weights are made as
//     2^(s - m + 15 - LAG4 - e), where 2^e, at least 2, is above every scale of a value so far: a weight and its product with a scale stay below 2^15, and small ones
//     above the last bit of f16 for 2^-34 of the largest.
//
// Copies are cp.async of 16 bytes a lane into a ring that no other warp sees, so nothing waits on a barrier; their places in it are such that no load has a bank conflict.
#pragma once

#include <cuda_runtime.h>

#include <cfloat>

#include "attend_join.cuh"
#include "attention.cuh"
#include "kernels.h"
#include "kv4_unpack.cuh"
#include "ptx.cuh"

namespace {

constexpr float LAG4 = 4.0f;

struct Attend4Params {
  AttnLayer a;
  KvBatchDev kv;
  const void *q;
  void *out;
  uint64_t q_stride, out_stride;
  AttnWorkspace ws;
  TileShape ts;
  uint32_t min_units;
  uint32_t page_units;  // 16 bytes between pages
  bool whole_pages;  // a chunk of 16 tokens lies in one page
};

// U: units of 32 values, GS: 1 where two units share a scale, NT: eights of rows.
template <int U, int GS, int NT>
struct Stream4Shape {
  static constexpr bool SMALL = U <= 4 && NT == 1;  // 128 registers a thread do
  static constexpr int NW = SMALL ? 4 : 4, CTAS = SMALL ? 4 : 2;
  static constexpr int G = (U + GS) >> GS, R = 8 * NT, TILES = 2 * U;
  static constexpr uint32_t KB = NW * 16, THREADS = NW * 32;
  static constexpr uint32_t CODES = 16 * 16 * U, SCALES = 16 * 4 * G, CHUNK = 2 * (CODES + SCALES);  // keys' codes and scales, values' codes and scales
  static constexpr int ST = U == 2 ? 6 : SMALL ? 4 : 5;
  static constexpr uint32_t RING = NW * ST * CHUNK, OP = 32 * U + 4;
  static constexpr uint32_t JOIN = NW * R * (OP + 2) * 4;  // the warps' maxima, sums and outputs
  static constexpr size_t SMEM = RING > JOIN ? RING : JOIN;
};

// Row of a chunk's token `t` among the columns of the scores: tokens j and j + 4 are neighbours, so that a lane's two tokens of values lie where no other's do.
__device__ __forceinline__ constexpr uint32_t slot_of(uint32_t t) { return (t & 8) | ((t & 3) << 1) | ((t >> 2) & 1); }
// Where 16-byte piece c of it lies among a token's.
template <int U>
__device__ __forceinline__ constexpr uint32_t key_piece(uint32_t slot, uint32_t c) {
  return U == 8 ? c ^ (slot & 1) : c;
}
template <int U>
__device__ __forceinline__ constexpr uint32_t value_piece(uint32_t t, uint32_t c) {
  return U == 8 ? c ^ ((t & 3) << 1) : U == 4 ? c ^ (t & 2) : c;
}

__device__ __forceinline__ void copy16_all(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(in ? N : 0) : "memory");
}
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

template <int U, int GS, int NT>
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
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, eighth = lane >> 2;
  const uint32_t D = p.a.head_dim, page_tokens = p.a.page_tokens, window = p.a.window;
  const bool f16 = p.a.cache_type == MER_VALUE_F16;
  const TileShape &ts = p.ts;
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
  // Where in a chunk the lane's pieces go: of codes, piece i * 32 + lane of the chunk's; of scales, lanes 0 .. 15 the keys', the others the values'.
  uint32_t k_to[(U + 1) / 2], v_to[(U + 1) / 2], scale_to = S::CODES + (lane < 16 ? 0 : S::CODES + S::SCALES) + slot_of(lane & 15) * (4 * G);
  const char *const scale_pages = (const char *)(lane < 16 ? p.kv.k_pages : p.kv.v_pages);
#pragma unroll
  for (int i = 0; i < (U + 1) / 2; i++) {
    const uint32_t e = i * 32 + lane, tok = e / U % 16, c = e % U, slot = slot_of(tok);
    k_to[i] = slot * (16 * U) + key_piece<U>(slot, c) * 16, v_to[i] = S::CODES + S::SCALES + tok * (16 * U) + value_piece<U>(tok, c) * 16;
    if (U == 4 && i) k_to[i] = k_to[0] + 512, v_to[i] = v_to[0] + 512;  // eight tokens on
    if (U == 4 ? i == 0 : true) asm volatile("" : "+r"(k_to[i]), "+r"(v_to[i]));  // kept, not made again for every chunk
  }
  asm volatile("" : "+r"(scale_to));

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
    // ---- the ring: the warp's blocks are b_lo .. b_hi, block b_lo + i lies in stage i % ST.  A lane knows the page of one token of a chunk, ST chunks ahead.
    const uint32_t w16 = warp * 16;
    const uint32_t b_lo = max(t.lo, start < w16 + 16 ? 0u : (start - w16 - 16) / KB + 1), b_hi = end <= w16 ? t.lo : min(t.hi, (end - w16 + KB - 1) / KB);
    // Blocks f_lo .. f_lo + f_n: whole chunks of one page each.
    const uint32_t f_lo = start <= w16 ? 0u : (start - w16 + KB - 1) / KB, f_hi = end < w16 + 16 || !p.whole_pages ? 0u : (end - w16 - 16) / KB + 1, f_n = min(f_hi, b_hi) > f_lo ? min(f_hi, b_hi) - f_lo : 0;
    const uint32_t *const table = p.kv.page_table + (uint64_t)t.seq * p.kv.table_stride;
    struct Place {
      uint32_t number, in;  // page, and the token in it (whole_pages: the chunk's first)
    };
    auto entry = [&](uint32_t blk) {
      const uint32_t key = blk * KB + w16 + (p.whole_pages ? 0 : lane & 15), slot = divided(key, p.kv.page_tokens);
      Place at;
      at.in = key - slot * page_tokens;
      at.number = blk < b_hi && (p.whole_pages || (key >= first_seen(t, window) && key < t.past + t.token0 + t.tokens)) && slot < p.kv.table_stride ? table[slot] : 0xFFFFFFFFu;
      return at;
    };
    const uint64_t head_at = t.kv_head * p.kv.head_stride;
    // in 16 bytes; scales in 4
    const uint64_t codes_at = head_at / 16 + lane, scales_at = (head_at + p.a.kv4.codes) / 4 + (lane & 15) * G;
    auto issue = [&](uint32_t blk, const Place &at, uint32_t stage) {
      constexpr int N = G % 4 == 0 ? 16 : G % 2 == 0 ? 8 : 4;
      const uint32_t dst = ring + stage * S::CHUNK;
      if (blk - f_lo < f_n && at.number < p.kv.n_pages) {
        const uint64_t page = (uint64_t)at.number * p.page_units;
        const uint64_t first = page + codes_at + at.in * U;
#pragma unroll
        for (int i = 0; i < (U + 1) / 2; i++) {
          if (U % 2 && i * 32 + lane >= 16 * U) continue;
          copy16_all(dst + k_to[i], (const char *)p.kv.k_pages + (first * 16 + i * 512));
          copy16_all(dst + v_to[i], (const char *)p.kv.v_pages + (first * 16 + i * 512));
        }
        const char *const src = scale_pages + (page * 16 + (scales_at + at.in * G) * 4);
#pragma unroll
        for (int i = 0; i < 4 * G / N; i++) {
          if constexpr (N == 16)
            copy16_all(dst + scale_to + i * N, src + i * N);
          else
            cp_async_small<N>(dst + scale_to + i * N, src + i * N, true);
        }
      } else if (blk < b_hi) {  // token by token; what it needs of the tile is read again
        const uint32_t end = t.past + t.token0 + t.tokens, start = first_seen(t, window);
        const uint32_t key = here(blk) * KB + w16 + (lane & 15), in = p.whole_pages ? here(at.in) + (lane & 15) : at.in;
        const bool seen = key >= start && key < end, there = seen && at.number < p.kv.n_pages;
        if (seen && !there) bad = 1;
        const uint64_t block = there ? at.number * p.kv.page_stride + t.kv_head * p.kv.head_stride : 0;
        const uint32_t valid = __ballot_sync(0xFFFFFFFFu, there);  // tokens of the chunk, twice
#pragma unroll
        for (int i = 0; i < (U + 1) / 2; i++) {
          const uint32_t e = i * 32 + here(lane), tok = e / U % 16, c = e % U;
          const uint64_t off = __shfl_sync(0xFFFFFFFFu, block, tok) + (uint64_t)__shfl_sync(0xFFFFFFFFu, in, tok) * (16 * U) + c * 16;
          if (U % 2 && e >= 16 * U) continue;
          const bool ok = valid >> tok & 1;
          copy16(dst + k_to[i], (const char *)p.kv.k_pages + (ok ? off : 0), ok ? 16 : 0);
          copy16(dst + v_to[i], (const char *)p.kv.v_pages + (ok ? off : 0), ok ? 16 : 0);
        }
        const char *const src = scale_pages + (there ? block + p.a.kv4.codes + (uint64_t)in * (4 * G) : 0);
#pragma unroll
        for (int i = 0; i < 4 * G / N; i++) {
          if constexpr (N == 16)
            copy16(dst + scale_to + i * N, src + (there ? i * N : 0), there ? 16 : 0);
          else
            cp_async_small<N>(dst + scale_to + i * N, src + (there ? i * N : 0), there);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    Place ahead[ST];
#pragma unroll
    for (int i = 0; i < ST; i++) ahead[i] = entry(b_lo + i);
    // ---- queries, before the copies: behind these they would wait for a full ring of every SM.  Lane (eighth, quad) has values 32 u + 8 quad .. of rows eighth and eighth + 8, as the
    // product's B operand wants them: pair p of the eight meets the codes from bits 4 p and 16 + 4 p on, which stand for themselves times 2^-24 where p is even, 2^-20 where it is odd.
    uint32_t qf[NT][U][4], qs[NT][(G + 3) / 4][2];  // qs: sums of a group's queries in two parts, each behind a zero
    float row_factor[NT];  // of row x * 8 + eighth
#pragma unroll
    for (int x = 0; x < NT; x++) {
      const uint32_t r = x * 8 + eighth, tok = r / t.heads, h = r - tok * t.heads;
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        raw[u] = make_uint4(0, 0, 0, 0);
        if (r < tile_rows && u * 32 + quad * 8 < D)
          raw[u] = *reinterpret_cast<const uint4 *>((const char *)p.q + ((uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + h) * D + u * 32 + quad * 8) * 2);
      }
      float top = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t w = e == 0 ? raw[u].x : e == 1 ? raw[u].y : e == 2 ? raw[u].z : raw[u].w;
          const float2 v = f16 ? __half22float2(as_half2(w)) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
          top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
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
          const uint32_t w = e == 0 ? raw[u].x : e == 1 ? raw[u].y : e == 2 ? raw[u].z : raw[u].w;
          float2 v = f16 ? __half22float2(as_half2(w)) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
          const __half2 n = __floats2half2_rn(v.x * per, v.y * per);
          v = __half22float2(n);
          sums[u >> GS] += v.x + v.y;
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
#pragma unroll
    for (int i = 0; i < ST - 1; i++) issue(b_lo + i, ahead[i], i);
    Place next_place = ahead[ST - 1];
    uint32_t stage = 0;
    // Every row sees the tokens all_from .. all_see; of the warp's chunks, those of blocks n_lo .. n_lo + n_n have no others.
    const uint32_t all_see = t.past + t.token0, all_from = window && end > window ? end - window : 0;
    const uint32_t n_lo = all_from <= w16 ? 0u : (all_from - w16 + KB - 1) / KB, n_hi = all_see < w16 + 15 ? 0u : (all_see - w16 - 15) / KB + 1, n_n = n_hi > n_lo ? n_hi - n_lo : 0;
    // The lane has rows x * 8 + quad * 2 + e of scores and outputs.  least: sums of weights times minima
    // A weight is 2^(s * factor - less) with less = m - shift; limit: the score from which on m has to follow, -infinity while there is no m.
    float o[NT][S::TILES][4], least[NT][4], less[NT][2], limit[NT][2], l[NT][2], factor[NT][2];
#pragma unroll
    for (int x = 0; x < NT; x++) {
#pragma unroll
      for (int e = 0; e < 2; e++) less[x][e] = 0.0f, limit[x][e] = -INFINITY, l[x][e] = 0.0f, factor[x][e] = __shfl_sync(0xFFFFFFFFu, row_factor[x], quad * 8 + e * 4);
#pragma unroll
      for (int e = 0; e < 4; e++) least[x][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < S::TILES; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[x][i][e] = 0.0f;
    }
    uint32_t room = 16;  // the exponent field of 2^e as an f16 has it
    for (uint32_t blk = b_lo; blk < b_hi; blk++) {
      {
        const Place at = next_place;
        next_place = entry(blk + ST);
        __syncwarp();  // the chunk that lay in this stage has been read
        issue(blk + ST - 1, at, stage == 0 ? ST - 1 : stage - 1);
      }
      const uint32_t base = ring + stage * S::CHUNK;
      stage = stage + 1 == ST ? 0 : stage + 1;
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
      __syncwarp();
      // ---- scores: s[x][T][e] of row x * 8 + quad * 2 + e and the token of slot T * 8 + eighth
      const uint32_t kscales = base + S::CODES, values = base + S::CODES + S::SCALES, vscales = values + S::CODES;
      float s[NT][2][2];
      {
        uint32_t words[2][U], sc[2][G];
#pragma unroll
        for (int T = 0; T < 2; T++) {
          const uint32_t row = base + (T * 8 + eighth) * (16 * U);
          if constexpr (U == 8) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint4 v = lds128(row + key_piece<U>(eighth, quad * 2 + i) * 16);
              words[T][4 * i] = v.x, words[T][4 * i + 1] = v.y, words[T][4 * i + 2] = v.z, words[T][4 * i + 3] = v.w;
            }
          } else {
            lds_words<U>(row + quad * (4 * U), words[T]);
          }
          lds_words<G>(kscales + (T * 8 + eighth) * (4 * G), sc[T]);
        }
        float mins[NT][4];
#pragma unroll
        for (int b = 0; b < (G + 3) / 4; b++) {
          uint32_t w[2];
#pragma unroll
          for (int T = 0; T < 2; T++) w[T] = b * 4 + quad < G ? lds32(kscales + (T * 8 + eighth) * (4 * G) + (b * 4 + quad) * 4) : 0u;
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
      if (blk - n_lo >= n_n) {
        const uint32_t at = here(blk) * KB + w16 + (eighth >> 1) + (eighth & 1) * 4;
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t last = t.past + t.token0 + min(x * 8 + quad * 2 + e, t.tokens * t.heads - 1) / t.heads;  // that the row sees
#pragma unroll
            for (int T = 0; T < 2; T++)
              if (!(at + T * 8 <= last && (window == 0 || at + T * 8 + window > last))) s[x][T][e] = -INFINITY;
          }
      }
      // ---- values' scales of the lane's tokens of slots T * 8 + quad * 2 and the next, by pairs
      uint32_t vs[2][G], any = 0;
#pragma unroll
      for (int T = 0; T < 2; T++) {
        uint32_t sc[2][G];
        lds_words<G>(vscales + (T * 8 + quad * 2) * (4 * G), sc[0]);
        lds_words<G>(vscales + (T * 8 + quad * 2 + 1) * (4 * G), sc[1]);
#pragma unroll
        for (int g = 0; g < G; g++) vs[T][g] = __byte_perm(sc[0][g], sc[1][g], 0x5410), any |= vs[T][g];
      }
      // ---- weights
      bool grows = (any & 0x40004000u) != 0;  // a scale of 2 or more
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int e = 0; e < 2; e++) grows |= fmaxf(s[x][0][e], s[x][1][e]) > limit[x][e];
      if (__any_sync(0xFFFFFFFFu, grows)) {
        uint32_t most = 0;
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
          for (int g = 0; g < G; g++) most = max(most, max(here(vs[T][g]) & 0x7FFFu, here(vs[T][g]) >> 16 & 0x7FFFu));  // numbers that are not negative have the order of their bits
        most = max((__reduce_max_sync(0xFFFFFFFFu, most) >> 10) + 1, room);  // the exponent of a power of two above them all
        const float was = 30.0f - LAG4 - (float)room, shift = 30.0f - LAG4 - (float)most, wider = __uint_as_float((127u + room - most) << 23);
        room = most;
#pragma unroll
        for (int x = 0; x < NT; x++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float top = fmaxf(s[x][0][e], s[x][1][e]);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            top *= factor[x][e];
            const bool first = limit[x][e] == -INFINITY;
            const float m = less[x][e] + was, now = first ? top : fmaxf(top, m), f = first ? 0.0f : exp2_approx(m - now) * wider;
            less[x][e] = now == -INFINITY ? 0.0f : now - shift;
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
      // ---- minima: row 2 g + 1 of the product (row g where a token's words are no whole 16 bytes) has group g's
      {
        uint32_t a0, a1 = 0, a2, a3 = 0;
        if constexpr (G % 4 == 0) {
          const uint32_t at = vscales + ((lane & 7) + (lane & 8)) * (4 * G) + (G == 8 ? (lane >> 4) * 16 : 0);
          if constexpr (G == 8)
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a0), "=r"(a2), "=r"(a1), "=r"(a3) : "r"(at) : "memory");
          else
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(a0), "=r"(a2) : "r"(at) : "memory");
        } else {
          const uint32_t at = vscales + quad * 2 * (4 * G) + (eighth % G) * 4;
          a0 = __byte_perm(lds32(at), lds32(at + 4 * G), 0x7632);
          a2 = __byte_perm(lds32(at + 8 * 4 * G), lds32(at + 9 * 4 * G), 0x7632);
        }
#pragma unroll
        for (int x = 0; x < NT; x++) mma_f16(least[x], a0, a1, a2, a3, pf[x][0], pf[x][1]);
      }
      // ---- values: a lane has words eighth * U .. of tokens quad, quad + 4, quad + 8 and quad + 12
      {
        uint32_t w[2][U];  // word u of the lane's two tokens, of 16 bits each
#pragma unroll
        for (int T = 0; T < 2; T++) {
          if constexpr (U == 3) {
#pragma unroll
            for (int u = 0; u < U; u++) {
              const uint32_t at = values + (T * 8 + quad) * (16 * U) + (eighth * U + u) * 2;
              w[T][u] = lds16(at) | lds16(at + 4 * 16 * U) << 16;
            }
          } else {
            uint32_t h[2][U / 2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
              const uint32_t tok = T * 8 + quad + 4 * b, byte = eighth * (2 * U);
              lds_words<U / 2>(values + tok * (16 * U) + value_piece<U>(tok, byte / 16) * 16 + byte % 16, h[b]);
            }
#pragma unroll
            for (int u = 0; u < U; u++) w[T][u] = __byte_perm(h[0][u / 2], h[1][u / 2], u % 2 ? 0x7632 : 0x5410);
          }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
          const uint32_t v0 = w[0][u] >> 8, v1 = w[1][u] >> 8;
#pragma unroll
          for (int x = 0; x < NT; x++) {
            const uint32_t b0 = as_u32(__hmul2(as_half2(pf[x][0]), as_half2(vs[0][u >> GS]))), b1 = as_u32(__hmul2(as_half2(pf[x][1]), as_half2(vs[1][u >> GS])));
            mma_f16(o[x][2 * u], w[0][u] & 0x000F000Fu, w[0][u] & 0x00F000F0u, w[1][u] & 0x000F000Fu, w[1][u] & 0x00F000F0u, b0, b1);
            mma_f16(o[x][2 * u + 1], v0 & 0x000F000Fu, v0 & 0x00F000F0u, v1 & 0x000F000Fu, v1 & 0x00F000F0u, b0, b1);
          }
        }
      }
    }
    // ---- the warps' results: [warp][row] reference and sum, [warp][row][OP] output, where the rings were
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
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
        const float l0 = __shfl_sync(0xFFFFFFFFu, least[x][at], src + quad), l1 = __shfl_sync(0xFFFFFFFFu, least[x][at + 1], src + quad);
        constexpr float LOW = 16777216.0f, HIGH = 1048576.0f;  // 2^24 and 2^20
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t row = x * 8 + quad * 2 + e;
          const float least_of = e ? l1 : l0;
          if (row < rows)
            *reinterpret_cast<float4 *>(s_o + ((size_t)warp * R + row) * S::OP + u * 32 + eighth * 4) =
                make_float4(fmaf(o[x][2 * u][e], LOW, least_of), fmaf(o[x][2 * u][2 + e], HIGH, least_of), fmaf(o[x][2 * u + 1][e], LOW, least_of), fmaf(o[x][2 * u + 1][2 + e], HIGH, least_of));
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
        for (uint32_t i = tid; i < rows * (DP / 4); i += THREADS) {
          const uint32_t r = i / (DP / 4), c = i % (DP / 4) * 4;
          float reference = -INFINITY, sum = 0.0f;
          float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
          for (uint32_t k = 0; k < n; k++) reference = fmaxf(reference, __ldcg(part_of_tile(run, t, p.ws.parts, c0, k, part_floats(R, DP)) + r));
#pragma unroll 4
          for (uint32_t k = 0; k < n; k++) {
            const float *from = part_of_tile(run, t, p.ws.parts, c0, k, part_floats(R, DP));
            const float mk = __ldcg(from + r), f = mk == -INFINITY ? 0.0f : exp2_approx(mk - reference);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(from + 2 * R + (size_t)r * DP + c));
            sum = fmaf(f, __ldcg(from + R + r), sum);
            acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
          }
          if (f16)
            store_row<__half>(p.a, t, r, c, reference, sum, acc, (__half *)p.out, p.out_stride);
          else
            store_row<__nv_bfloat16>(p.a, t, r, c, reference, sum, acc, (__nv_bfloat16 *)p.out, p.out_stride);
        }
      }
    }
    __syncthreads();  // the rings are copied into again
  }
  if (bad) atomicOr(p.ws.status, MER_DEVSTAT_BAD_CACHE);
}

template <int U, int GS, int NT>
cudaError_t launch_stream4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws, int sm_count, cudaStream_t s) {
  using S = Stream4Shape<U, GS, NT>;
  const Attend4Params p{a, kv, q, out, q_stride, out_stride, ws, TileShape(a.q_heads, a.kv_heads, S::R, ATTEND4_START, 1, 0, ATTEND4_WHOLE), ATTEND4_MIN_RUN, (uint32_t)(kv.page_stride / 16), a.page_tokens % 16 == 0};
  const cudaError_t e = allow_smem<k_attend4<U, GS, NT>>(S::SMEM);
  if (e != cudaSuccess) return e;
  return launch_overlapped(k_attend4<U, GS, NT>, dim3(sm_count * S::CTAS), S::THREADS, S::SMEM, s, false, p);
}

}  // namespace
