// A cache that holds keys and values in 4 bits: where the bytes of a page lie.  A page of one key head is a block: the codes of its tokens one behind the other,
// then their scales and minima.
//
//   x stands as the code clamp(rint((x - minimum) / scale), 0, 15) and for scale * code + minimum; `group` neighbouring values of a head share scale and minimum.
//
// A head's codes are stored for 64, 96, 128, 192 or 256 values, `units` of 32 (what is behind the head's own values: zeros), 16 bytes a unit.  The orders are the
// matrix units' own, so that a lane's operand is one load:
//   keys    32-bit word j * units + u (j < 4): values 32 u + 8 j + 2 p and + 2 p + 1 from bits 4 p and 16 + 4 p on (p < 4)
//   values  16-bit word r * units + u (r < 8): values 32 u + 4 r + i from bit 4 i on (i < 4)
// Scale and minimum of a group are two f16, side by side.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define KV4_HD __host__ __device__ __forceinline__
#else
#define KV4_HD inline
#endif

// What a key's value is off by at most when norm and rotation are made in 32 bits, as a share of the largest value M of its head.  In units of 2^-24, with r the size of a pair (a, b)
// that is turned, times norm's weights, r <= sqrt(2) M, and |a| + |b| <= sqrt(2) r <= 2 M:
//   an angle of at most a half-turn rounded, 2^-25 of it: pi / 2 r              2.23
//   cosine and sine, 1 unit in the last place below 1 as CUDA states: |a| + |b|   2
//   they times rope_scale and times a weight: r each                            2.83
//   the first of the two products: at most r                                    1.42
//   their sum: M                                                                1
//   the norm: a lane's four sums of squares, its halves, five exchanges (heads above 128 values), f32(1 / head_dim), the sum with eps: 12, of which the root takes half    6
//   rsqrtf, 2 units in the last place as CUDA states, each up to 2^-23 of the value    4
//   the product with it                                                         1
// together 20.5, held as 24: a cosine of two units in the last place has room, too.
constexpr float KV4_KEY_ERROR = 0x1.8p-20f;

struct Kv4Shape {
  uint32_t group, units, groups;  // values that share a scale (32 or 64), stored units of 32 values, stored groups
  uint32_t codes;                 // bytes of a block's codes
  KV4_HD uint32_t token_bytes() const { return 16 * units; }
  KV4_HD uint32_t scale_bytes() const { return 4 * groups; }
};
inline uint32_t kv4_units(uint32_t head_dim) { return head_dim <= 64 ? 2 : head_dim <= 96 ? 3 : head_dim <= 128 ? 4 : head_dim <= 192 ? 6 : 8; }
inline Kv4Shape kv4_shape(uint32_t head_dim, uint32_t page_tokens, uint32_t group) {
  Kv4Shape s;
  s.group = group, s.units = kv4_units(head_dim);
  s.groups = (32 * s.units + group - 1) / group;
  s.codes = page_tokens * s.token_bytes();
  return s;
}
// Bytes of a block, a whole number of 16.
inline uint64_t kv4_block_bytes(const Kv4Shape &s, uint32_t page_tokens) { return (s.codes + (uint64_t)page_tokens * s.scale_bytes() + 15) / 16 * 16; }
// What the kernels rely on of a cache's pages (strides in bytes); null when they can be run.
inline const char *kv4_pages_fault(const Kv4Shape &s, uint32_t page_tokens, uint32_t kv_heads, uint32_t n_pages, uint64_t page_stride, uint64_t token_stride, uint64_t head_stride) {
  if (token_stride) return "a cache of 4 bits has no token stride: the tokens of a page's head lie in its block";
  if ((page_stride | head_stride) % 16) return "page and head strides must be multiples of 16 bytes";
  const uint64_t block = kv4_block_bytes(s, page_tokens), most = 1ull << 47;
  if ((kv_heads > 1 && head_stride < block) || (n_pages > 1 && page_stride < block)) return "a stride is smaller than a head's block";
  if (page_stride >> 36 || head_stride >> 36) return "pages or heads lie 64 GB or more apart";
  if ((n_pages > 1 && page_stride > most / (n_pages - 1)) || (kv_heads > 1 && head_stride > most / (kv_heads - 1))) return "keys or values reach over more than 2^47 bytes";
  return nullptr;
}
