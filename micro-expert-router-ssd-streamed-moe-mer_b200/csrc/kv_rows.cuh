// Vectors of a row's values on their way through registers.
#pragma once

#include "attention.cuh"

namespace {

// V values as they lie in memory.
template <typename T, int V>
struct Raw {
  static constexpr int BYTES = sizeof(T) * V;
  __align__(16) T t[V];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; i++) reinterpret_cast<uint4 *>(t)[i] = *(reinterpret_cast<const uint4 *>(p) + i);
    } else if constexpr (BYTES == 8) {
      reinterpret_cast<uint2 *>(t)[0] = *reinterpret_cast<const uint2 *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) t[i] = p[i];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < BYTES / 2; i++) reinterpret_cast<uint16_t *>(t)[i] = 0;
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = Num<T>::f(t[i]);
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[V]) {
  if constexpr (V % 2 == 0) {
    uint32_t t[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) t[i] = Num<T>::pack(x[2 * i], x[2 * i + 1]);
    if constexpr (V == 8)
      *reinterpret_cast<uint4 *>(p) = make_uint4(t[0], t[1], t[2], t[3]);
    else
      *reinterpret_cast<uint2 *>(p) = make_uint2(t[0], t[1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = Num<T>::one(x[i]);
  }
}
// Whether `v` values of `size` bytes from `p`, `stride` apart, can be moved as one vector.
inline bool vec_ok(const void *p, uint64_t stride, uint32_t v, uint32_t size) {
  const uint32_t bytes = v * size < 16 ? v * size : 16;
  return p == nullptr || ((uintptr_t)p % bytes == 0 && stride * size % bytes == 0);
}

}  // namespace
