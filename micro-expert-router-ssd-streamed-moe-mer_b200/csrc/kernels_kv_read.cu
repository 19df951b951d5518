// Keys and values of a batch's rows out of the pages, as rows of numbers: for a prefix that is handed on, another kernel, or a look at what a cache holds.
//
//   16-bit cache: the value itself;  4 bits: scale * code + minimum, one fma in fp32 (the product has 15 bits);  one rounding to the rows' type.
//
// What bounds it: memory.  A lane has a part of a token's head that is one piece of its bytes: four units' words of a key or a value (32 values of a head of 128; its scales are
// one vector more), or eight 16-bit values.  A warp takes some rows one behind the other, which mostly follow one another in a sequence, so that their place is
// looked up once and their pages' numbers are one load; the lanes share out the rows' parts, and the loads of two parts are in flight before the first is stored.
// 32000 rows of 2 x 4 heads of 128 out of 4 bits to bf16, groups of 32: 18.4 us, 71 % of the measured copy's rate (a lane eight values, a row looked up for itself: 33); 64 rows 6.8, the call on the host.
// To f32 L1 bounds it (74 % busy): a lane's eight values are two stores of 16 bytes, each half of 32 neighbouring ones; 13411 rows of 2 x 8 heads of 80 23.6 us for 12.1 of bytes.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "kernels.h"
#include "kv4_unpack.cuh"
#include "ptx.cuh"

namespace {

constexpr uint32_t READ_THREADS = 128, READ_ROWS = 8;

struct ReadParams {
  AttnLayer a;
  KvBatchDev kv;
  KvRowsDev r;
  uint32_t *status;
  uint32_t rows;   // of a warp, at most 32
  uint32_t parts;  // of a head
  FastDiv by_parts;
  bool vec;        // rows are whole vectors of 16 bytes
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

// Eight codes: of a word of a key, pair i from bits 4 i and 16 + 4 i on; of two words of a value, the same bits of the first half and of the second are values i and i + 4.
__device__ __forceinline__ void eight_codes(uint32_t w, __half2 (&n)[4]) {
  const __half2 whole = as_half2(0x64006400u), sixteenth = as_half2(0x2C002C00u), back = as_half2(0xD400D400u);  // 1024, 1 / 16, -64
  const uint32_t v = w >> 8;
  n[0] = __hsub2(as_half2((w & 0x000F000Fu) | 0x64006400u), whole), n[1] = __hfma2(as_half2((w & 0x00F000F0u) | 0x64006400u), sixteenth, back);
  n[2] = __hsub2(as_half2((v & 0x000F000Fu) | 0x64006400u), whole), n[3] = __hfma2(as_half2((v & 0x00F000F0u) | 0x64006400u), sixteenth, back);
}

// N words from an address on a multiple of 4 N (at most 16) bytes.
template <int N>
__device__ __forceinline__ void load_words(const char *p, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1) {
    if constexpr (N % 4 == 0) {
      const uint4 v = *reinterpret_cast<const uint4 *>(p + i * 4);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    } else if constexpr (N % 2 == 0) {
      const uint2 v = *reinterpret_cast<const uint2 *>(p + i * 4);
      w[i] = v.x, w[i + 1] = v.y;
    } else {
      w[i] = *reinterpret_cast<const uint32_t *>(p + i * 4);
    }
  }
}

// A part of a token's head on its way: U units' words of a cache of 4 bits, or (U == 0) eight 16-bit values.
template <typename CACHE, int U>
struct Part {
  uint32_t words[U ? U : 4], scales[U ? U : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t &w : words) w = 0;
#pragma unroll
    for (uint32_t &w : scales) w = 0;
  }
  // `token`: the first of the head's bytes of the token; part `j`
  __device__ __forceinline__ void load(const char *token, const char *token_scales, uint32_t j, bool wide) {
    if constexpr (U == 0) {
      load_words<4>(token + j * 16, words);
    } else {
      load_words<U>(token + j * (4 * U), words);
      if (wide) {
        uint32_t g[(U + 1) / 2];
        load_words<(U + 1) / 2>(token_scales, g);
#pragma unroll
        for (int u = 0; u < U; u++) scales[u] = g[u / 2];
      } else {
        load_words<U>(token_scales, scales);
      }
    }
  }
  template <typename OUT>
  __device__ __forceinline__ void store(OUT *head, uint32_t j, uint32_t head_dim, bool key, bool vec) const {
    float x[8];
    if constexpr (U == 0) {
      const CACHE *const t = reinterpret_cast<const CACHE *>(words);
#pragma unroll
      for (int v = 0; v < 8; v++) x[v] = Num<CACHE>::f(t[v]);
      store_eight<OUT>(head + j * 8, x, vec);
    } else {
      // words u of 16 bits of a value's rows 2 j and 2 j + 1 are the halves u and U + u of the part
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (u * 32 + j * 8 >= head_dim) break;
        const float scale = __low2float(as_half2(scales[u])), least = __high2float(as_half2(scales[u]));
        const uint32_t w = key ? words[u] : __byte_perm(words[u / 2], words[(U + u) / 2], (u % 2 ? 0x32u : 0x10u) | ((U + u) % 2 ? 0x7600u : 0x5400u));
        __half2 code[4];
        eight_codes(w, code);
        float y[4][2];
#pragma unroll
        for (int v = 0; v < 4; v++) y[v][0] = fmaf(scale, __low2float(code[v]), least), y[v][1] = fmaf(scale, __high2float(code[v]), least);
#pragma unroll
        for (int v = 0; v < 8; v++) x[v] = key ? y[v / 2][v % 2] : y[v % 4][v / 4];
        store_eight<OUT>(head + u * 32 + j * 8, x, vec);
      }
    }
  }
};

// CACHE: the pages' type where they hold 16 bits (U == 0).
template <typename CACHE, int U, typename OUT>
__global__ void __launch_bounds__(READ_THREADS) k_kv_read(const __grid_constant__ ReadParams p) {
  const Kv4Shape &f = p.a.kv4;
  const uint32_t lane = threadIdx.x & 31, warp = blockIdx.x * (READ_THREADS / 32) + threadIdx.x / 32;
  grid_dep_wait();
  grid_dep_launch();
  const uint64_t first = (uint64_t)warp * p.rows;
  if (first >= p.kv.n_rows) return;
  const uint32_t row0 = (uint32_t)first, n_rows = min(p.rows, p.kv.n_rows - row0);
  // Lane r has row r's page and the token in it; ~0: none, zeros, ~1: the row belongs to no sequence.
  uint32_t page = 0xFFFFFFFFu, in_page = 0;
  for (uint32_t r = 0; r < n_rows;) {
    RowPlace at;
    if (!find_row(p.kv, p.a.page_tokens, row0 + r, lane, &at)) {
      if (lane == r++) page = 0xFFFFFFFEu;
      continue;
    }
    // Rows r .. last of its sequence have a place if the first one has; one without is looked up alone.
    const uint32_t last = at.first == 0xFFFFFFFFu ? r + 1 : min(n_rows, at.end - row0);
    if (at.first != 0xFFFFFFFFu && lane >= r && lane < last) {
      const uint32_t pos = at.first + (lane - r), slot = divided(pos, p.kv.page_tokens);
      const uint32_t number = slot < p.kv.table_stride ? p.kv.page_table[(uint64_t)at.seq * p.kv.table_stride + slot] : 0xFFFFFFFFu;
      page = number < p.kv.n_pages ? number : 0xFFFFFFFFu;
      in_page = pos - slot * p.a.page_tokens;
    }
    r = last;
  }
  if (lane < n_rows && page == 0xFFFFFFFFu) atomicOr(p.status, MER_DEVSTAT_BAD_CACHE);
  // Item e of the warp's: part e % parts of head (e / parts) % kv_heads of the keys, then of the values, of the rows one behind the other.
  const uint32_t per_row = 2 * p.a.kv_heads * p.parts, items = n_rows * per_row;
  uint32_t key_or_value, head, j, row = 0, e = lane;  // of the item; rows are counted, not divided
  const auto locate = [&](uint32_t in_row) {
    const uint32_t h = divided(in_row, p.by_parts);
    j = in_row - h * p.parts;
    key_or_value = h >= p.a.kv_heads, head = key_or_value ? h - p.a.kv_heads : h;
  };
  uint32_t in_row = lane;
  for (; e - lane < items; e += 64) {
    Part<CACHE, U> part[2];
    OUT *dst[2];
    uint32_t js[2];
    bool keys[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
      while (in_row >= per_row) in_row -= per_row, row++;
      const uint32_t number = __shfl_sync(0xFFFFFFFFu, page, row & 31), in = __shfl_sync(0xFFFFFFFFu, in_page, row & 31);
      locate(in_row);
      js[b] = j, keys[b] = !key_or_value;
      OUT *const rows = (OUT *)(key_or_value ? p.r.v : p.r.k);
      dst[b] = row < n_rows && number != 0xFFFFFFFEu && rows ? rows + (uint64_t)(row0 + row) * (key_or_value ? p.r.v_stride : p.r.k_stride) + head * p.a.head_dim : nullptr;
      part[b].clear();
      if (dst[b] && number != 0xFFFFFFFFu) {
        const char *const pages = (const char *)(key_or_value ? p.kv.v_pages : p.kv.k_pages);
        if constexpr (U != 0) {
          const char *const block = pages + number * p.kv.page_stride + head * p.kv.head_stride;
          part[b].load(block + in * (16 * U), block + f.codes + in * f.scale_bytes(), j, f.group == 64);
        } else {
          part[b].load(pages + (number * p.kv.page_stride + in * p.kv.token_stride + head * p.kv.head_stride) * sizeof(CACHE), nullptr, j, false);
        }
      }
      in_row += 32;
    }
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (dst[b]) part[b].store(dst[b], js[b], p.a.head_dim, keys[b], p.vec);
  }
}

template <typename CACHE, int U>
cudaError_t launch_read(const ReadParams &p, uint32_t grid, cudaStream_t s) {
  return p.r.type == MER_VALUE_F32   ? launch_overlapped(k_kv_read<CACHE, U, float>, dim3(grid), READ_THREADS, 0, s, false, p)
         : p.r.type == MER_VALUE_F16 ? launch_overlapped(k_kv_read<CACHE, U, __half>, dim3(grid), READ_THREADS, 0, s, false, p)
                                     : launch_overlapped(k_kv_read<CACHE, U, __nv_bfloat16>, dim3(grid), READ_THREADS, 0, s, false, p);
}

}  // namespace

cudaError_t launch_kv_read(const AttnLayer &a, const KvBatchDev &kv, const KvRowsDev &r, uint32_t *status, int sm_count, cudaStream_t s) {
  ReadParams p{a, kv, r, status};
  p.parts = a.q4 ? 4 : a.head_dim / 8, p.by_parts = fast_div(p.parts);
  const uint32_t size = r.type == MER_VALUE_F32 ? 4 : 2;
  p.vec = ((uintptr_t)r.k | (uintptr_t)r.v | (r.k ? r.k_stride * size : 0) | (r.v ? r.v_stride * size : 0)) % 16 == 0;
  // Rows of a warp: several where there are more than fill the machine.
  p.rows = (uint32_t)std::min<uint64_t>(READ_ROWS, std::max<uint64_t>(1, kv.n_rows / ((uint64_t)sm_count * 32)));
  const uint64_t warps = ((uint64_t)kv.n_rows + p.rows - 1) / p.rows;
  const uint32_t grid = (uint32_t)((warps + READ_THREADS / 32 - 1) / (READ_THREADS / 32));  // below 2^31: n_rows is
  if (!a.q4) return a.cache_type == MER_VALUE_F16 ? launch_read<__half, 0>(p, grid, s) : launch_read<__nv_bfloat16, 0>(p, grid, s);
  switch (a.kv4.units) {
    case 2: return launch_read<uint8_t, 2>(p, grid, s);
    case 3: return launch_read<uint8_t, 3>(p, grid, s);
    case 4: return launch_read<uint8_t, 4>(p, grid, s);
    case 6: return launch_read<uint8_t, 6>(p, grid, s);
    default: return launch_read<uint8_t, 8>(p, grid, s);
  }
}
