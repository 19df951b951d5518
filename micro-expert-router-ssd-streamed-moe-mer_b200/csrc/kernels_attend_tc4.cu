// Attention of many new rows over a paged cache of 4 bits: attend_tc.cuh, whose copying warps unpack (attend_tc4.cuh).
#include "attend_tc.cuh"

namespace {

template <typename IO>
cudaError_t launch_tc4(const TcParams &p, int sm_count, cudaStream_t s) {
  const TcMaps none{};
  switch (p.a.kv4.units) {
    case 2: return launch_tc<IO, 64, 2>(p, none, sm_count, s);
    case 3: return launch_tc<IO, 128, 3>(p, none, sm_count, s);
    case 4: return launch_tc<IO, 128, 4>(p, none, sm_count, s);
    case 6: return launch_tc<IO, 256, 6>(p, none, sm_count, s);
    default: return launch_tc<IO, 256, 8>(p, none, sm_count, s);
  }
}

}  // namespace

cudaError_t launch_attend_tc4(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                              int sm_count, cudaStream_t s) {
  const TcParams p = tc_params(a, kv, q, q_stride, out, out_stride, ws);
  return a.cache_type == MER_VALUE_F16 ? launch_tc4<__half>(p, sm_count, s) : launch_tc4<__nv_bfloat16>(p, sm_count, s);
}
