// Attention of a few new tokens a sequence over a paged cache of 4 bits: attend4.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <stdint.h>

namespace {
// The cut of a batch into runs; 32 and 4 heads of 128, us.  START 2, 4, 8: 64 tokens behind 800 to 8000 49.5, 48.7, 52.1.  WHOLE 2, 6, 12: one token behind 32000 23.0, 23.2, 26.8, the
// 64 tokens alike.  MIN_RUN 2 and 6: both alike, so the longer one, whose parts are fewer.
constexpr uint32_t ATTEND4_WHOLE = 6;    // blocks of a tile that is not cut
constexpr uint32_t ATTEND4_START = 4;    // what a tile costs beside its blocks, in blocks
constexpr uint32_t ATTEND4_MIN_RUN = 6;  // units of the shortest run
}  // namespace

#include "attend4.cuh"

namespace {

template <int GS, int NT>
cudaError_t launch_stream4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws, int sm_count, cudaStream_t s) {
  switch (a.kv4.units) {
    case 2: return launch_stream4<2, GS, NT>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
    case 3: return launch_stream4<3, GS, NT>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
    case 4: return launch_stream4<4, GS, NT>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
    case 6: return launch_stream4<6, GS, NT>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
    default: return launch_stream4<8, GS, NT>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
  }
}

}  // namespace

size_t attend4_part_floats(int sm_count) { return sm_count * ATTEND4_SM_FLOATS; }

cudaError_t launch_attend4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws, int sm_count,
                           cudaStream_t s) {
  // Up to eight query heads of a key head: eight rows a tile, else sixteen, whose registers leave half as many warps (8 drafts of 5 tokens and 4 heads 44 us with eight, 51 with sixteen).
  const bool few = a.q_heads / a.kv_heads <= 8;
  if (a.kv4.group == 32)
    return few ? launch_stream4<0, 1>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s) : launch_stream4<0, 2>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
  return few ? launch_stream4<1, 1>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s) : launch_stream4<1, 2>(a, kv, q, q_stride, out, out_stride, ws, sm_count, s);
}
