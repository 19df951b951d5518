// Keys and values of a batch's rows out of the pages, as rows of numbers: for a prefix that is handed on, another kernel, or a look at what a cache holds.
//
//   16-bit cache: the value itself;  4 bits: scale * code + minimum, one fma in fp32 (the product has 15 bits);  one rounding to the rows' type.
//
// What bounds it: memory.  A lane has eight neighbouring values of a head (a word of codes and its group's scale and minimum in, one or two 16-byte vectors out); a
// warp takes some rows one behind the other, which mostly follow one another in a sequence, so that their place is looked up once and their pages' numbers are one load.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace {

constexpr uint32_t READ_THREADS = 128;
constexpr int READ_AT_ONCE = 4;  // items of a lane in flight

struct ReadParams {
  AttnLayer a;
  KvBatchDev kv;
  KvRowsDev r;
  uint32_t *status;
  uint32_t rows;      // of a warp, at most 32
  uint32_t pieces;    // eights of a head
  FastDiv by_pieces;
  uint32_t items;     // of a row: keys, then values
  bool vec;           // rows are whole vectors of 16 bytes
};

template <typename OUT>
__device__ __forceinline__ void store_eight(OUT *p, const float (&x)[8], bool vec) {
  if constexpr (sizeof(OUT) == 4) {
    if (vec) {
      reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
      return;
    }
  } else if (vec) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(Num<OUT>::pack(x[0], x[1]), Num<OUT>::pack(x[2], x[3]), Num<OUT>::pack(x[4], x[5]), Num<OUT>::pack(x[6], x[7]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) p[i] = Num<OUT>::one(x[i]);
}

// CACHE: the pages' type, or uint8_t where they hold 4 bits.
template <typename CACHE, typename OUT>
__global__ void __launch_bounds__(READ_THREADS) k_kv_read(const ReadParams p) {
  constexpr bool Q4 = sizeof(CACHE) == 1;
  const AttnLayer &a = p.a;
  const Kv4Shape &f = a.kv4;
  const uint32_t lane = threadIdx.x & 31, warp = blockIdx.x * (READ_THREADS / 32) + threadIdx.x / 32;
  grid_dep_wait();
  grid_dep_launch();
  const uint64_t row0 = (uint64_t)warp * p.rows;
  if (row0 >= p.kv.n_rows) return;
  const uint32_t behind = (uint32_t)min((uint64_t)p.kv.n_rows, row0 + p.rows), per_part = a.kv_heads * p.pieces;
  RowPlace at;
  at.end = 0;
  uint32_t numbers = 0, first = 0;  // the lanes have the page numbers of the rows from `first` on
  for (uint32_t row = (uint32_t)row0; row < behind; row++) {
    bool placed = row < at.end;  // the same sequence as the row before
    if (!placed) {
      if (!find_row(p.kv, a.page_tokens, row, lane, &at)) continue;
      first = row;
      if (at.pos != 0xFFFFFFFFu) {
        const uint32_t slot = divided(at.pos + lane, p.kv.page_tokens);
        numbers = row + lane < min(at.end, behind) && slot < p.kv.table_stride ? p.kv.page_table[(uint64_t)at.seq * p.kv.table_stride + slot] : 0xFFFFFFFFu;
      } else {
        at.end = row + 1;  // the next row is looked up again: it may have a place
      }
    }
    uint32_t page = 0xFFFFFFFFu, in_page = 0;
    if (at.pos != 0xFFFFFFFFu) {
      const uint32_t pos = at.pos + (row - first);
      page = __shfl_sync(0xFFFFFFFFu, numbers, row - first);
      in_page = pos - divided(pos, p.kv.page_tokens) * a.page_tokens;
    }
    const bool held = page < p.kv.n_pages;
    if (!held && lane == 0) atomicOr(p.status, MER_DEVSTAT_BAD_CACHE);
    for (uint32_t i0 = lane; i0 < p.items; i0 += 32 * READ_AT_ONCE) {
      float x[READ_AT_ONCE][8];
      OUT *dst[READ_AT_ONCE];
      uint4 raw[READ_AT_ONCE];
      uint32_t scale_min[READ_AT_ONCE];
      bool key[READ_AT_ONCE];
#pragma unroll
      for (int n = 0; n < READ_AT_ONCE; n++) {
        const uint32_t i = i0 + n * 32;
        key[n] = i < per_part;
        const uint32_t e = key[n] ? i : i - per_part, head = divided(e, p.by_pieces), piece = e - head * p.pieces;
        OUT *rows = (OUT *)(key[n] ? p.r.k : p.r.v);
        dst[n] = i < p.items && rows ? rows + row * (key[n] ? p.r.k_stride : p.r.v_stride) + head * a.head_dim + piece * 8 : nullptr;
        raw[n] = make_uint4(0, 0, 0, 0), scale_min[n] = 0;
        if (!dst[n] || !held) continue;
        const char *pages = (const char *)(key[n] ? p.kv.k_pages : p.kv.v_pages);
        if constexpr (Q4) {
          const char *block = pages + page * p.kv.page_stride + head * p.kv.head_stride;
          const char *codes = block + (uint64_t)in_page * f.token_bytes();
          const uint32_t u = piece / 4, j = piece % 4;
          if (key[n]) {
            raw[n].x = *reinterpret_cast<const uint32_t *>(codes + (j * f.units + u) * 4);
          } else {
            raw[n].x = *reinterpret_cast<const uint16_t *>(codes + (2 * j * f.units + u) * 2);
            raw[n].y = *reinterpret_cast<const uint16_t *>(codes + ((2 * j + 1) * f.units + u) * 2);
          }
          scale_min[n] = *reinterpret_cast<const uint32_t *>(block + f.codes + (uint64_t)in_page * f.scale_bytes() + piece * 8 / f.group * 4);
        } else {
          raw[n] = *reinterpret_cast<const uint4 *>((const CACHE *)pages + page * p.kv.page_stride + (uint64_t)in_page * p.kv.token_stride + head * p.kv.head_stride + piece * 8);
        }
      }
#pragma unroll
      for (int n = 0; n < READ_AT_ONCE; n++) {
        if constexpr (Q4) {
          const __half2 h = *reinterpret_cast<const __half2 *>(&scale_min[n]);
          const float scale = __low2float(h), least = __high2float(h);
#pragma unroll
          for (int v = 0; v < 8; v++) {
            const uint32_t code = key[n] ? raw[n].x >> (v / 2 * 4 + v % 2 * 16) & 15 : (v < 4 ? raw[n].x : raw[n].y) >> (v % 4 * 4) & 15;
            x[n][v] = fmaf(scale, (float)code, least);
          }
        } else {
          const CACHE *t = reinterpret_cast<const CACHE *>(&raw[n]);
#pragma unroll
          for (int v = 0; v < 8; v++) x[n][v] = Num<CACHE>::f(t[v]);
        }
        if (dst[n]) store_eight<OUT>(dst[n], x[n], p.vec);
      }
    }
  }
}

template <typename CACHE>
cudaError_t launch_read(const ReadParams &p, uint32_t grid, cudaStream_t s) {
  return p.r.type == MER_VALUE_F32   ? launch_overlapped(k_kv_read<CACHE, float>, dim3(grid), READ_THREADS, 0, s, false, p)
         : p.r.type == MER_VALUE_F16 ? launch_overlapped(k_kv_read<CACHE, __half>, dim3(grid), READ_THREADS, 0, s, false, p)
                                     : launch_overlapped(k_kv_read<CACHE, __nv_bfloat16>, dim3(grid), READ_THREADS, 0, s, false, p);
}

}  // namespace

cudaError_t launch_kv_read(const AttnLayer &a, const KvBatchDev &kv, const KvRowsDev &r, uint32_t *status, int sm_count, cudaStream_t s) {
  ReadParams p{a, kv, r, status};
  p.pieces = a.head_dim / 8, p.by_pieces = fast_div(p.pieces), p.items = 2 * a.kv_heads * p.pieces;
  const uint32_t size = r.type == MER_VALUE_F32 ? 4 : 2;
  p.vec = ((uintptr_t)r.k | (uintptr_t)r.v | (r.k ? r.k_stride * size : 0) | (r.v ? r.v_stride * size : 0)) % 16 == 0;
  // Rows of a warp: several where there are more than fill the machine.
  p.rows = (uint32_t)std::min<uint64_t>(8, std::max<uint64_t>(1, kv.n_rows / ((uint64_t)sm_count * 32)));
  const uint64_t warps = ((uint64_t)kv.n_rows + p.rows - 1) / p.rows, ctas = (warps + READ_THREADS / 32 - 1) / (READ_THREADS / 32);
  const uint32_t grid = (uint32_t)ctas;  // below 2^31: n_rows is
  return a.cache_type == MER_VALUE_F16 && !a.q4 ? launch_read<__half>(p, grid, s) : !a.q4 ? launch_read<__nv_bfloat16>(p, grid, s) : launch_read<uint8_t>(p, grid, s);
}
