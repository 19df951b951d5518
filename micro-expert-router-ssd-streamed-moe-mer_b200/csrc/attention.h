// Internal interface of the attention side of a layer: constants of a layer, a batch over the paged cache, launchers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kv4.h"

// Division of numbers below 2^31 by a constant of a launch: multiplier and shift of Granlund and Montgomery, "Division by invariant integers using
// multiplication" (1994), section 4; below 2^31 its last sum has room in 32 bits.
struct FastDiv {
  uint32_t mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f{0, 0};
  while ((1ull << f.shift) < d) f.shift++;
  f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
  return f;
}

// One installed layer (mer_attention_install); the pointers are device memory, parts of `constants`.
struct AttnLayer {
  uint32_t q_heads, kv_heads, head_dim, page_tokens;
  uint32_t window;                // tokens that a row sees, itself among them; 0 = all before it
  float scale;                    // of the scores
  int cache_type;                 // MER_VALUE_F16 or MER_VALUE_BF16: queries, outputs, and the cache where it does not hold 4 bits
  bool q4;                        // keys and values in 4 bits, as kv4 says
  Kv4Shape kv4;
  uint32_t rope_dims;             // leading values of a head that are rotated
  int rope_pairs;                 // neighbours instead of halves
  float rope_scale, norm_eps;
  const float *q_norm, *k_norm;   // [head_dim] or null
  const double *turns;            // [rope_dims / 2] half turns per position: frequency / pi
  const float *sinks;             // [q_heads] or null
  void *constants;
};

// A token's place in the pages as a 32-bit number of 16-byte pieces.
#define KV_MAX_SPAN (((1ull << 32) - 1) * 8)

// mer_kv_batch as the kernels take it.
struct KvBatchDev {
  void *k_pages, *v_pages;
  uint64_t page_stride, token_stride, head_stride;  // in values; all places lie below KV_MAX_SPAN.  In 4 bits: in bytes, and no token_stride
  FastDiv page_tokens;
  uint32_t capacity;  // tokens that a row of the table has pages for
  const uint32_t *page_table, *row_start, *kv_len;
  uint32_t n_pages, table_stride, n_seqs, n_rows;
  uint32_t least_rows = 0, most_rows = 0xFFFFFFFFu;  // the sequences that an attention kernel sees to bring so many rows
};

struct QkvRowsDev {
  const void *q, *k, *v;
  void *q_out;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;  // in values
  int type;
};

// kernels_kv.cu
cudaError_t launch_kv_append(const AttnLayer &a, const KvBatchDev &kv, const QkvRowsDev &rows, uint32_t *status, int sm_count, cudaStream_t s);

// kernels_kv4.cu: the same for a cache of 4 bits
cudaError_t launch_kv4_append(const AttnLayer &a, const KvBatchDev &kv, const QkvRowsDev &rows, uint32_t *status, int sm_count, cudaStream_t s);

// Rows that keys and values are read back to; either may be null.
struct KvRowsDev {
  void *k, *v;
  uint64_t k_stride, v_stride;  // in values
  int type;
};
// kernels_kv_read.cu
cudaError_t launch_kv_read(const AttnLayer &a, const KvBatchDev &kv, const KvRowsDev &rows, uint32_t *status, int sm_count, cudaStream_t s);

// Workspace of the attention kernels: `parts` floats and `counts` zeroed words that every call leaves zero.
struct AttnWorkspace {
  float *parts;
  uint32_t *counts, *status;
};
size_t attend_part_floats(int sm_count);
// kernels_attend_tc.cu
size_t attend_tc_part_floats(int sm_count);
cudaError_t launch_attend_tc(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                             int sm_count, cudaStream_t s);
// kernels_attend_tc4.cu
cudaError_t launch_attend_tc4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                              int sm_count, cudaStream_t s);
// kernels_attend4.cu
constexpr uint32_t ATTEND_CTAS = 2;  // an SM's at most, of any attention kernel: a count each, and two parts
size_t attend4_part_floats(int sm_count);
cudaError_t launch_attend4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws, int sm_count,
                           cudaStream_t s);
// kernels_attend.cu
size_t attend_counts(int sm_count);
cudaError_t launch_attend(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                          int sm_count, cudaStream_t s, int *launches);
