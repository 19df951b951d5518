// Codes of a cache of 4 bits as f16 numbers in registers.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "kv4.h"

namespace {

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t *>(&v); }

// The eight codes of a word, times scale, plus minimum: pair i has the codes from bits 4 i and 16 + 4 i on.  A code is put into the mantissa of 1024 (or, sixteen times
// as large, where it stands), from which it comes out exactly; the last fma rounds once, 2^-11 of the value at most.
// (Published for integer weights by Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022; the constants are f16's.)
__device__ __forceinline__ uint4 kv4_numbers(uint32_t w, __half2 scale, __half2 least) {
  const __half2 whole = as_half2(0x64006400u), sixteenth = as_half2(0x2C002C00u), back = as_half2(0xD400D400u);  // 1024, 1 / 16, -64
  const uint32_t v = w >> 8;
  uint4 x;
  x.x = as_u32(__hfma2(__hsub2(as_half2((w & 0x000F000Fu) | 0x64006400u), whole), scale, least));
  x.y = as_u32(__hfma2(__hfma2(as_half2((w & 0x00F000F0u) | 0x64006400u), sixteenth, back), scale, least));
  x.z = as_u32(__hfma2(__hsub2(as_half2((v & 0x000F000Fu) | 0x64006400u), whole), scale, least));
  x.w = as_u32(__hfma2(__hfma2(as_half2((v & 0x00F000F0u) | 0x64006400u), sixteenth, back), scale, least));
  return x;
}
// Values are unpacked from two 16-bit words of four: value v of the eight stands at this place.
__host__ __device__ constexpr int kv4_value_at(int v) { return v < 4 ? 2 * v : 2 * (v - 4) + 1; }

}  // namespace
