// The rows of a layer's q|k|v projection on their way into attention over a cache of 4 bits, one pass: RMSNorm of every query and key head, position rotation, queries out in
// their type, keys and values quantised into the pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w;   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * frequency_j
//   minimum = f16(min y), scale = f16(f32(max y - min y) * f32(1 / 15)), unit = f32(1 / scale) or 0, code = clamp(rint((y - minimum) * unit), 0, 15)
//
// over groups of 32 or 64 neighbouring values of a key or value head.  A lane has eight neighbouring values of a head, one 32-bit word of codes; the eight that they rotate with it
// loads beside them (the other lane's own, so from L1), which leaves groups whole in neighbouring lanes whatever is rotated with what.  What a key is multiplied by, cosine and norm's
// weight in one, stays in registers through a row's heads.
// Codes, scales and minima are those of 64-bit arithmetic: 32 bits would give a value next to the border between two codes the other one about once in a million values, and a minimum next to
// one between two f16 would take its whole group's codes with it.  So a step of keys or values is made in 32 bits with a bound on its error; where anything of it lies within that bound
// of a border (one step of keys in nine with two heads of 128 a step, one in seventeen with one), it is made again in 64.  A group with a value that is not finite, or beyond KV4_MOST, which f16 has no room for, has the minimum NaN: all of it reads back as NaN.
// Queries: angles in half turns reduced in 64 bits, the rest in 32, one rounding at the end.
//
// What bounds it: issuing.  A step of queries is 111 instructions, one of keys and one of values 598 together, a warp 950 beside its steps.  Captured calls, us: prompt of 2048 rows of
// 32 + 2 x 4 heads of 128, bf16, 17.0 (16-bit cache: 10.0); 13411 rows of 32 + 2 x 8 heads of 80 in f16 85 at 58 % of the issue slots; one token 4.2.  With their rows read back
// the 13411 rows took 244 us with keys and values wholly in 64 bits, 125 with values in 32, 112 so.  No faster: CTAs of four warps, four an SM; two warps to every row.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "attention.cuh"
#include "kernels.h"
#include "kv_rows.cuh"
#include "pack2.cuh"
#include "ptx.cuh"

namespace {

constexpr uint32_t WARPS = 16;

struct Kv4Params {
  AttnLayer a;
  KvBatchDev kv;
  QkvRowsDev r;
  uint32_t *status;
  uint32_t lanes;             // of a head, a power of two
  uint32_t q_steps, kv_steps; // steps of 32 / lanes heads: of the queries, of the keys and as many of the values
  uint32_t chunks, each;      // warps of a row, and steps of each
  bool vec;                   // rows by vectors of 8 values
  bool q_vec;                 // queries out by vectors of 8 values
  float per_value;            // 1 / head_dim
  double per_value64;
};

constexpr float KV4_MOST = 60000.0f;

// The nearest of the sixteen, of t = (x - minimum) * unit in 64 bits: 1.5 * 2^52 leaves the nearest whole number in the sum's low bits.
__device__ __forceinline__ uint32_t kv4_code(double t) { return (uint32_t)__vimin_s32_relu(__double2loint(t + 6755399441055744.0), 15); }

struct Kv4Group {
  uint32_t scale_min;  // f16, f16
  float unit, from;
};
// Of a group's least and largest value; `range`: their difference, rounded once.
__device__ __forceinline__ Kv4Group kv4_group(float lo, float range, bool odd) {
  const __half least = __float2half_rn(lo), scale = __float2half_rn(__fmul_rn(range, 1.0f / 15.0f));
  const float s = __half2float(scale);
  Kv4Group g;
  g.scale_min = odd ? 0x7E000000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(least) << 16;
  g.unit = s > 0.0f && !odd ? __frcp_rn(s) : 0.0f, g.from = odd ? 0.0f : __half2float(least);  // odd: codes of zero
  return g;
}
// Whether any lane of this one's group says so.
__device__ __forceinline__ bool kv4_any(bool v, uint32_t lane, uint32_t lanes) {
  return (__ballot_sync(0xFFFFFFFFu, v) & ((lanes == 8 ? 0xFFu : 0xFu) << (lane & ~(lanes - 1)))) != 0;
}

// Codes of a key's eight values, and its group's scale and minimum; `there`: the lane has values.
__device__ __forceinline__ uint32_t kv4_key_codes(const double (&y)[8], bool there, uint32_t lane, uint32_t lanes, uint32_t (&code)[8]) {
  double lo = INFINITY, hi = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    odd |= !(fabs(y[i]) <= (double)KV4_MOST);
    lo = y[i] < lo ? y[i] : lo, hi = y[i] > hi ? y[i] : hi;
  }
  if (!there) odd = false, lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (uint32_t d = 1; d < 8; d *= 2) {
    if (d >= lanes) break;
    const double l = __shfl_xor_sync(0xFFFFFFFFu, lo, d), h = __shfl_xor_sync(0xFFFFFFFFu, hi, d);
    lo = l < lo ? l : lo, hi = h > hi ? h : hi;
  }
  const Kv4Group g = kv4_group((float)lo, (float)(hi - lo), kv4_any(odd, lane, lanes));
  const double unit = g.unit, from = g.from;
#pragma unroll
  for (int i = 0; i < 8; i++) code[i] = kv4_code(g.unit == 0.0f ? 0.0 : (y[i] - from) * unit);  // also of what is no number
  return g.scale_min;
}
// A key's eight values in 32 bits, each off by at most `error` from what 64 bits have: codes and their group's scale and minimum, or false where a border is too near for that.
__device__ __forceinline__ bool kv4_key_codes_fast(const float (&y)[8], float error, bool there, uint32_t lanes, uint32_t (&code)[8], uint32_t *scale_min) {
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; i++) lo = fminf(lo, y[i]), hi = fmaxf(hi, y[i]);
  if (!there) lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (uint32_t d = 1; d < 8; d *= 2) {
    if (d >= lanes) break;
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d)), hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
  }
  const float range = hi - lo, more = 2.25f * error;  // range, at most twice the head's largest value, is rounded by a twelfth of error at most; the other roundings keep the order
  const __half least = __float2half_rn(lo - error), scale = __float2half_rn((range - more) * (1.0f / 15.0f));
  bool sure = __half_as_ushort(least) == __half_as_ushort(__float2half_rn(lo + error)) && __half_as_ushort(scale) == __half_as_ushort(__float2half_rn((range + more) * (1.0f / 15.0f)));
  *scale_min = (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(least) << 16;
  const float s = __half2float(scale), unit = s > 0.0f ? __frcp_rn(s) : 0.0f, from = __half2float(least);
  float near = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float t = (y[i] - from) * unit, r = t + 12582912.0f;  // 1.5 * 2^23
    near = fmaxf(near, fabsf(t - (r - 12582912.0f)));
    code[i] = (uint32_t)__vimin_s32_relu(__float_as_int(r) - 0x4B400000, 15);
  }
  sure = sure && near <= 0.5f - 0x1p-18f - error * unit;
  return sure || !there;
}
// The same of values, which are 32-bit numbers as they come.  t in 32 bits is off by at most 2^-24 of t, of the difference, and of the product: below 2^-18 where a code is
// below 16, so only a t that near the border between two codes is made again in 64.
__device__ __forceinline__ uint32_t kv4_value_codes(const float (&x)[8], bool there, uint32_t lane, uint32_t lanes, uint32_t (&code)[8]) {
  float lo = INFINITY, hi = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    odd |= !(fabsf(x[i]) <= KV4_MOST);
    lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
  }
  if (!there) odd = false, lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (uint32_t d = 1; d < 8; d *= 2) {
    if (d >= lanes) break;
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d)), hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
  }
  const Kv4Group g = kv4_group(lo, hi - lo, kv4_any(odd, lane, lanes));
  float near = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float t = (x[i] - g.from) * g.unit, r = t + 12582912.0f;  // 1.5 * 2^23
    near = fmaxf(near, fabsf(t - (r - 12582912.0f)));
    code[i] = (uint32_t)__vimin_s32_relu(__float_as_int(r) - 0x4B400000, 15);
  }
  if (g.unit == 0.0f) {
#pragma unroll
    for (uint32_t &c : code) c = 0;  // also of what is no number
  } else if (near > 0.5f - 0x1p-18f) {  // or a t beyond 2^22, which is no code
#pragma unroll
    for (int i = 0; i < 8; i++) code[i] = kv4_code(((double)x[i] - (double)g.from) * (double)g.unit);
  }
  return g.scale_min;
}

// What steps cost, in steps of queries (by instructions): a row's steps are cut into equal runs of these.
constexpr uint32_t K_COST = 4, V_COST = 2;
// The first step whose beginning is not before unit x of a row's.
__host__ __device__ inline uint32_t kv4_step_at(uint32_t x, uint32_t q_steps, uint32_t kv_steps) {
  if (x <= q_steps) return x;
  x -= q_steps;
  if (x <= K_COST * kv_steps) return q_steps + (x + K_COST - 1) / K_COST;
  return q_steps + kv_steps + (x - K_COST * kv_steps + V_COST - 1) / V_COST;
}

// IN: the rows' type, OUT: the queries'.
// PAIRS: neighbours rotate into one another.
template <typename IN, typename OUT, bool PAIRS>
__global__ void __launch_bounds__(32, 16) k_kv4_append(const __grid_constant__ Kv4Params p) {
  extern __shared__ double2 turns[];  // [rope_dims / 2] cosine and sine
  const AttnLayer &a = p.a;
  const Kv4Shape &f = a.kv4;
  const uint32_t lane = threadIdx.x, row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  const uint32_t D = a.head_dim, half = a.rope_dims / 2, U = f.units;
  const uint32_t sub = lane & (p.lanes - 1), heads = 32 / p.lanes, of = lane / p.lanes, d0 = sub * 8;
  const bool there = d0 < D, stored = sub < 4 * U;
  // Steps: queries, keys, values.
  const uint32_t k_first = p.q_steps, v_first = k_first + p.kv_steps, steps = v_first + p.kv_steps;
  const uint32_t first = min(steps, kv4_step_at(chunk * p.each, p.q_steps, p.kv_steps)), end = min(steps, kv4_step_at((chunk + 1) * p.each, p.q_steps, p.kv_steps));
  // what value d0 + i rotates with: its number, or its own
  auto mate = [&](uint32_t v) { return v >= a.rope_dims ? v : PAIRS ? v ^ 1 : v < half ? v + half : v - half; };
  const bool has_mate = there && !PAIRS && d0 < a.rope_dims;  // in another lane
  const int mate_at = has_mate ? (int)mate(d0) - (int)d0 : 0;
  // The lane's eight values of a head, and their mates.
  auto ask = [&](const IN *src, Raw<IN, 8> &x, Raw<IN, 8> &y, bool mates) {
    if (p.vec) {
      x.load(src);
      if (mates) y.load(src + mate_at);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x.t[e] = src[e];
      if (mates) {
#pragma unroll
        for (int e = 0; e < 8; e++) y.t[e] = src[(int)mate(d0 + e) - (int)d0];
      }
    }
  };
  constexpr int AHEAD = sizeof(IN) == 2 ? 3 : 2;  // steps of queries whose values are on their way
  Raw<IN, 8> own[AHEAD], other[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) own[i].clear(), other[i].clear();  // what is never asked for stays zero
  const IN *const q_row = (const IN *)p.r.q + row * p.r.q_stride + of * D + d0;
  auto ask_query = [&](uint32_t step, Raw<IN, 8> &x, Raw<IN, 8> &y) {
    if (step < min(end, k_first) && there && step * heads + of < a.q_heads) ask(q_row + step * (heads * D), x, y, has_mate);
  };
  auto ask_key = [&](uint32_t step, Raw<IN, 8> &x, Raw<IN, 8> &y) {
    const uint32_t head = (step - k_first) * heads + of;
    if (step < min(end, v_first) && there && head < a.kv_heads) ask((const IN *)p.r.k + row * p.r.k_stride + head * D + d0, x, y, has_mate);
  };
  auto ask_value = [&](uint32_t step, Raw<IN, 8> &x) {
    const uint32_t head = (step - v_first) * heads + of;
    if (step < end && there && head < a.kv_heads) ask((const IN *)p.r.v + row * p.r.v_stride + head * D + d0, x, x, false);
  };
  grid_dep_wait();
  grid_dep_launch();
  if (first < k_first) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++) ask_query(first + i, own[i], other[i]);
  } else if (first < v_first) {
    ask_key(first, own[0], other[0]);
  } else {
    ask_value(first, own[0]);
  }
  RowPlace at;
  if (!find_row(p.kv, a.page_tokens, row, lane, &at)) return;
  if (at.pos == 0xFFFFFFFFu) {
    if (lane == 0) atomicOr(p.status, MER_DEVSTAT_BAD_CACHE);
    return;
  }
  uint32_t step = first;
  float2 *const turns32 = reinterpret_cast<float2 *>(turns + half);  // [rope_dims / 2] the same in 32 bits
  auto half_turns = [&](uint32_t i) {
    const double x = (double)at.pos * __ldg(a.turns + i);
    return x - 2.0 * rint(0.5 * x);
  };
  if (first < min(end, v_first)) {
    for (uint32_t i = lane; i < half; i += 32) {
      float sin, cos;
      sincospif((float)half_turns(i), &sin, &cos);
      turns32[i] = make_float2(cos * a.rope_scale, sin * a.rope_scale);
    }
    __syncwarp();
  }
  // What value i and its mate are multiplied by.
  auto factors = [&](const float *norm, const auto *table, auto(&cw)[8], auto(&sw)[8]) {
    using F = typename std::remove_reference<decltype(cw[0])>::type;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t v = d0 + i;
      cw[i] = (F)1, sw[i] = (F)0;
      if (v < a.rope_dims) {
        const auto t = table[PAIRS ? v / 2 : v < half ? v : v - half];
        cw[i] = (F)t.x, sw[i] = (F)((PAIRS ? v % 2 == 0 : v < half) ? -t.y : t.y);
      }
      if (norm && there) cw[i] *= (F)__ldg(norm + v), sw[i] *= (F)__ldg(norm + mate(v));
    }
  };
  // Norm and rotation of eight values in 32 bits.  Returned: what the norm multiplies by.
  auto turned = [&](const float(&x)[8], const float(&o)[8], const float(&cw)[8], const float(&sw)[8], bool norm, float(&z)[8]) -> float {
    float unit = 1.0f;
    uint64_t y[4], sq = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint64_t x2 = pack2(x[2 * e], x[2 * e + 1]), o2 = PAIRS ? pack2(x[2 * e + 1], x[2 * e]) : pack2(o[2 * e], o[2 * e + 1]);
      y[e] = fma2(o2, pack2(sw[2 * e], sw[2 * e + 1]), mul2(x2, pack2(cw[2 * e], cw[2 * e + 1])));
      sq = fma2(x2, x2, sq);
    }
    if (norm) {
      float lo, hi;
      unpack2(sq, lo, hi);
      lo += hi;
#pragma unroll
      for (uint32_t d = 1; d < 8; d *= 2) lo += __shfl_xor_sync(0xFFFFFFFFu, lo, d);
      if (p.lanes > 8) lo += __shfl_xor_sync(0xFFFFFFFFu, lo, 8);
      if (p.lanes > 16) lo += __shfl_xor_sync(0xFFFFFFFFu, lo, 16);
      unit = rsqrtf(fmaf(lo, p.per_value, a.norm_eps));
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = mul2(y[e], pack2(unit, unit));
    }
#pragma unroll
    for (int e = 0; e < 4; e++) unpack2(y[e], z[2 * e], z[2 * e + 1]);
    return unit;
  };
  // ---- queries
  if (step < min(end, k_first)) {
    const uint32_t q_end = min(end, k_first);
    float cw[8], sw[8];
    factors(a.q_norm, turns32, cw, sw);
    OUT *const to = (OUT *)p.r.q_out + row * p.r.q_out_stride + of * D + d0;
    auto rotate = [&](Raw<IN, 8> &mine, Raw<IN, 8> &theirs) {
      float x[8], o[8], z[8];
      mine.get(x), theirs.get(o);
      ask_query(step + AHEAD, mine, theirs);
      turned(x, o, cw, sw, a.q_norm != nullptr, z);
      __syncwarp();  // q may be rotated in place: all that is asked for of these heads has come
      if (there && step * heads + of < a.q_heads) {
        OUT *const dst = to + step * (heads * D);
        if (p.q_vec) {
          store_vec<OUT, 8>(dst, z);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) dst[e] = Num<OUT>::one(z[e]);
        }
      }
      step++;
    };
    while (step < q_end) {
#pragma unroll
      for (int i = 0; i < AHEAD; i++)
        if (step < q_end) rotate(own[i], other[i]);
    }
    own[0].clear(), other[0].clear();
    if (end > k_first) ask_key(k_first, own[0], other[0]);
  }
  const uint32_t lanes = f.group / 8, u = sub / 4, j = sub % 4;
  const uint64_t page = at.page * p.kv.page_stride, codes_at = page + at.in_page * f.token_bytes(), scales_at = page + f.codes + at.in_page * f.scale_bytes() + sub / lanes * 4;
  // ---- keys
  if (step < min(end, v_first)) {
    const uint32_t k_end = min(end, v_first);
    bool have64 = false;  // the table in 64 bits
    float cw[8], sw[8];
    factors(a.k_norm, turns32, cw, sw);
    uint8_t *const to = (uint8_t *)p.kv.k_pages + codes_at + (j * U + u) * 4, *const scale_to = (uint8_t *)p.kv.k_pages + scales_at;
#pragma unroll 1
    for (; step < k_end; step++) {
      const uint32_t head = (step - k_first) * heads + of;
      const Raw<IN, 8> mine = own[0], theirs = other[0];
      own[0].clear(), other[0].clear();
      if (step + 1 < v_first)
        ask_key(step + 1, own[0], other[0]);
      else
        ask_value(step + 1, own[0]);
      uint32_t code[8], scale_min;
      bool sure;
      {
        float x[8], o[8], z[8];
        mine.get(x), theirs.get(o);
        const float unit = turned(x, o, cw, sw, a.k_norm != nullptr, z);
        // off by KV4_KEY_ERROR of the head's largest value at most.  No square is infinite, and none that counts has lost bits, while their mean lies between 2^-96 and 2^120; what
        // other numbers lose below 2^-126 is times `unit` at most.
        float most = fmaxf(fmaxf(fmaxf(fabsf(z[0]), fabsf(z[1])), fmaxf(fabsf(z[2]), fabsf(z[3]))), fmaxf(fmaxf(fabsf(z[4]), fabsf(z[5])), fmaxf(fabsf(z[6]), fabsf(z[7]))));
        const float sum = ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));  // what is no number stays none
#pragma unroll
        for (uint32_t d = 1; d < 8; d *= 2) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
        if (p.lanes > 8) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 8));
        if (p.lanes > 16) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 16));
        sure = kv4_key_codes_fast(z, fmaf(most, KV4_KEY_ERROR, FLT_MIN * fmaxf(unit, 1.0f)), there, lanes, code, &scale_min) && most < 0.98f * KV4_MOST && sum - sum == 0.0f &&
               unit > 0x1p-60f && unit < 0x1p48f;
      }
      // A head that does not exist is zeros, whose least value may have either sign: nothing of it is stored, so it asks for nothing.  (An existing head of zeros does; its minimum has 64 bits' sign.)
      if (!__all_sync(0xFFFFFFFFu, sure || head >= a.kv_heads)) {
        if (!have64) {
          for (uint32_t i = lane; i < half; i += 32) {
            double2 t;
            sincospi(half_turns(i), &t.y, &t.x);
            turns[i] = make_double2(t.x * (double)a.rope_scale, t.y * (double)a.rope_scale);
          }
          __syncwarp();
          have64 = true;
        }
        double cw64[8], sw64[8], y[8], z[8];
        factors(a.k_norm, turns, cw64, sw64);
        float x[8], o[8];
        mine.get(x), theirs.get(o);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (double)x[e];
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = fma(PAIRS ? y[e ^ 1] : (double)o[e], sw64[e], y[e] * cw64[e]);
        if (a.k_norm) {
          double sq = 0.0;
#pragma unroll
          for (int e = 0; e < 8; e++) sq = fma(y[e], y[e], sq);
#pragma unroll 1
          for (uint32_t d = 1; d < p.lanes; d *= 2) sq += __shfl_xor_sync(0xFFFFFFFFu, sq, d);
          const double unit = rsqrt(fma(sq, p.per_value64, (double)a.norm_eps));
#pragma unroll
          for (int e = 0; e < 8; e++) z[e] *= unit;
        }
        scale_min = kv4_key_codes(z, there, lane, lanes, code);
      }
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) w += code[e] << (e / 2 * 4 + e % 2 * 16);
      if (stored && head < a.kv_heads) {
        const uint64_t head_at = head * p.kv.head_stride;
        *reinterpret_cast<uint32_t *>(to + head_at) = there ? w : 0u;
        if (sub % lanes == 0) *reinterpret_cast<uint32_t *>(scale_to + head_at) = there ? scale_min : 0u;
      }
    }
  }
  // ---- values
  uint8_t *const pages = (uint8_t *)p.kv.v_pages + codes_at, *const scale_to = (uint8_t *)p.kv.v_pages + scales_at;
  const uint32_t r = 2 * j;
#pragma unroll 1
  for (; step < end; step++) {
    const uint32_t head = (step - v_first) * heads + of;
    float x[8];
    own[0].get(x);
    own[0].clear();
    ask_value(step + 1, own[0]);
    uint32_t code[8];
    const uint32_t scale_min = kv4_value_codes(x, there, lane, lanes, code);
    uint32_t w0 = code[0] + (code[1] << 4) + (code[2] << 8) + (code[3] << 12), w1 = code[4] + (code[5] << 4) + (code[6] << 8) + (code[7] << 12);
    if (!there) w0 = w1 = 0;
    // words of unit u and the next one lie side by side: the lanes that have both exchange one of theirs
    const uint32_t given = __shfl_xor_sync(0xFFFFFFFFu, u % 2 ? w0 : w1, 4);
    if (stored && head < a.kv_heads) {
      const uint64_t head_at = head * p.kv.head_stride;
      if (U % 2 == 0) {
        *reinterpret_cast<uint32_t *>(pages + head_at + ((r + u % 2) * U + (u & ~1u)) * 2) = u % 2 ? given | w1 << 16 : w0 | given << 16;
      } else {
        *reinterpret_cast<uint16_t *>(pages + head_at + (r * U + u) * 2) = (uint16_t)w0;
        *reinterpret_cast<uint16_t *>(pages + head_at + ((r + 1) * U + u) * 2) = (uint16_t)w1;
      }
      if (sub % lanes == 0) *reinterpret_cast<uint32_t *>(scale_to + head_at) = there ? scale_min : 0u;
    }
  }
}

template <typename IN>
cudaError_t launch_kv4(const Kv4Params &p, uint32_t grid, size_t smem, cudaStream_t s) {
  if (p.a.cache_type == MER_VALUE_F16)
    return p.a.rope_pairs ? launch_overlapped(k_kv4_append<IN, __half, true>, dim3(grid), 32, smem, s, false, p)
                          : launch_overlapped(k_kv4_append<IN, __half, false>, dim3(grid), 32, smem, s, false, p);
  return p.a.rope_pairs ? launch_overlapped(k_kv4_append<IN, __nv_bfloat16, true>, dim3(grid), 32, smem, s, false, p)
                        : launch_overlapped(k_kv4_append<IN, __nv_bfloat16, false>, dim3(grid), 32, smem, s, false, p);
}

}  // namespace

cudaError_t launch_kv4_append(const AttnLayer &a, const KvBatchDev &kv, const QkvRowsDev &r, uint32_t *status, int sm_count, cudaStream_t s) {
  Kv4Params p{a, kv, r, status, 1};
  const uint32_t in = r.type == MER_VALUE_F32 ? 4 : 2;
  while (p.lanes < 4 * a.kv4.units) p.lanes *= 2;
  const uint32_t heads = 32 / p.lanes;
  p.q_steps = r.q ? (a.q_heads + heads - 1) / heads : 0, p.kv_steps = (a.kv_heads + heads - 1) / heads;
  p.vec = vec_ok(r.q, r.q_stride, 8, in) && vec_ok(r.k, r.k_stride, 8, in) && vec_ok(r.v, r.v_stride, 8, in) && (a.rope_pairs || a.rope_dims % 16 == 0);
  p.q_vec = vec_ok(r.q_out, r.q_out_stride, 8, 2);
  p.per_value64 = 1.0 / a.head_dim, p.per_value = (float)p.per_value64;
  // A warp a row, and more of them while there are fewer than WARPS an SM: fewer steps one after the other.
  const uint32_t units = p.q_steps + (K_COST + V_COST) * p.kv_steps;
  p.chunks = (uint32_t)std::min<uint64_t>(p.q_steps + 2 * p.kv_steps, std::max<uint64_t>(1, (uint64_t)sm_count * WARPS / kv.n_rows));
  p.each = (units + p.chunks - 1) / p.chunks;
  p.chunks = (units + p.each - 1) / p.each;
  const uint32_t grid = kv.n_rows * p.chunks;  // one row's warps only where rows are few: below 2^31
  const size_t smem = (size_t)(a.rope_dims / 2) * (sizeof(double2) + sizeof(float2));
  return r.type == MER_VALUE_F32 ? launch_kv4<float>(p, grid, smem, s) : r.type == MER_VALUE_F16 ? launch_kv4<__half>(p, grid, smem, s) : launch_kv4<__nv_bfloat16>(p, grid, smem, s);
}
