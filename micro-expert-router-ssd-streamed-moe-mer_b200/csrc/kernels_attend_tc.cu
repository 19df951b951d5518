// Attention of many new rows over a paged cache of 16-bit values: attend_tc.cuh.
#include "attend_tc.cuh"

namespace {

template <typename T>
cudaError_t launch_tc(const TcParams &p, const TcMaps &maps, int sm_count, cudaStream_t s) {
  if (p.a.head_dim <= 64) return launch_tc<T, 64, 0>(p, maps, sm_count, s);
  return p.a.head_dim <= 128 ? launch_tc<T, 128, 0>(p, maps, sm_count, s) : launch_tc<T, 256, 0>(p, maps, sm_count, s);
}

}  // namespace

size_t attend_tc_part_floats(int sm_count) { return (size_t)2 * sm_count * std::max(part_floats(TcShape<128, 0>::R, 128), part_floats(TcShape<256, 0>::R, 256)); }

cudaError_t launch_attend_tc(const AttnLayer &a, const KvBatchDev &kv, const void *q, uint64_t q_stride, void *out, uint64_t out_stride, const AttnWorkspace &ws,
                             int sm_count, cudaStream_t s) {
  const PageMapShape m(a, kv, TC_KB);
  TcMaps maps{};
  TcParams p = tc_params(a, kv, q, q_stride, out, out_stride, ws);
  p.box = encode_page_maps(&maps.pages, m, a, kv) ? m.rows : 0, p.head_first = m.head_first;
  p.q_mapped = p.ts.chunks == 1 && encode_row_map(&maps.q, q, a, kv.n_rows, q_stride, p.ts.heads, p.ts.tokens);
  return a.cache_type == MER_VALUE_F16 ? launch_tc<__half>(p, maps, sm_count, s) : launch_tc<__nv_bfloat16>(p, maps, sm_count, s);
}
