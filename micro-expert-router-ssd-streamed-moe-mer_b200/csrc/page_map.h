// Tensor maps over the pages of a cache, for tiled copies of runs of tokens.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mer_b200.h"
#include "attention.h"

// A page as the encoder sees it: [page][token][head][value], or tokens and heads the other way round, whichever makes the strides rise.
struct PageMapShape {
  uint64_t dims[4], strides[3];  // strides in bytes
  uint32_t box[4];
  uint32_t rows;    // tokens of a copy, 0: no map
  bool head_first;  // dimension 1 is the head

  // Copies of up to `most` tokens (a power of two).  A copy is a whole number of 8-row swizzle atoms and stays in its page, so only pages of a
  // multiple of 8 tokens have a map; and only such whose strides the encoder's description allows: each a multiple of the one before, and no
  // smaller than what lies within it.
  PageMapShape(const AttnLayer &a, const KvBatchDev &kv, uint32_t most) : dims{}, strides{}, box{}, rows(0), head_first(true) {
    uint32_t r = most;
    while (a.page_tokens % r) r /= 2;
    if (r < 8) return;
    uint64_t head = kv.head_stride * 2, token = kv.token_stride * 2, page = kv.page_stride * 2;
    head_first = a.page_tokens == 1 || a.kv_heads == 1 || head <= token;
    uint64_t n1 = head_first ? a.kv_heads : a.page_tokens, n2 = head_first ? a.page_tokens : a.kv_heads;
    uint64_t s1 = head_first ? head : token, s2 = head_first ? token : head;
    // a dimension of one has no stride of its own
    if (n1 == 1) s1 = (uint64_t)a.head_dim * 2;
    if (n2 == 1) s2 = s1 * n1;
    if (kv.n_pages == 1) page = s2 * n2;
    if (s1 < (uint64_t)a.head_dim * 2 || s2 < s1 * n1 || page < s2 * n2 || s2 % s1 || page % s2 || page >= (1ull << 40)) return;
    dims[0] = a.head_dim, dims[1] = n1, dims[2] = n2, dims[3] = kv.n_pages;
    strides[0] = s1, strides[1] = s2, strides[2] = page;
    box[0] = 64, box[1] = head_first ? 1 : r, box[2] = head_first ? r : 1, box[3] = 1;
    rows = r;
  }
};

// Keys and values; what lies beyond a head's values or behind the last page reads as zeros.
struct PageMaps {
  CUtensorMap k, v;
};
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once; null when the driver has none.
inline EncodeTiledFn page_map_encoder() {
  static const EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
  }();
  return fn;
}
inline bool encode_map(CUtensorMap *map, const AttnLayer &a, const void *base, uint32_t rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
  const EncodeTiledFn fn = page_map_encoder();
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return fn && fn(map, a.cache_type == MER_VALUE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(base), dims, strides, box,
                  step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// False where these pages have no map: then rows are copied one by one.
inline bool encode_page_maps(PageMaps *maps, const PageMapShape &m, const AttnLayer &a, const KvBatchDev &kv) {
  if (m.rows == 0) return false;
  const cuuint64_t dims[4] = {m.dims[0], m.dims[1], m.dims[2], m.dims[3]}, strides[3] = {m.strides[0], m.strides[1], m.strides[2]};
  const cuuint32_t box[4] = {m.box[0], m.box[1], m.box[2], m.box[3]};
  return encode_map(&maps->k, a, kv.k_pages, 4, dims, strides, box) && encode_map(&maps->v, a, kv.v_pages, 4, dims, strides, box);
}
// Rows of heads, `heads` of `rows` rows at a time.
inline bool encode_row_map(CUtensorMap *map, const void *base, const AttnLayer &a, uint32_t n_rows, uint64_t stride, uint32_t heads, uint32_t rows) {
  if (stride % a.head_dim) return false;
  const cuuint64_t dims[3] = {a.head_dim, a.q_heads, n_rows}, strides[2] = {a.head_dim * 2ull, stride * 2};
  const cuuint32_t box[3] = {64, heads, rows};
  return encode_map(map, a, base, 3, dims, strides, box);
}
