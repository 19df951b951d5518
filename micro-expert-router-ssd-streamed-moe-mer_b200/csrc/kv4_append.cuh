// Keys and values of a row on their way into a cache of 4 bits.  Included by kernels_kv.cu, for the warps of its kernel that have them.
//
//   minimum = f16(min x), scale = f16(f32(max x - min x) * f32(1 / 15)), unit = f32(1 / scale) or 0, code = clamp(rint((x - minimum) * unit), 0, 15)
//
// over groups of 32 or 64 neighbouring values.  A lane has eight neighbouring values of a head, one 32-bit word of codes, and loads the eight that they rotate with
// beside them.  Norm, rotation and codes are 64-bit arithmetic: a value next to the border between two codes, or a minimum next to one between two f16, gets the
// definition's, where 32 bits would give another one about once in a million values and move a whole group's codes with its minimum.
// A group with a value that is not finite, or beyond KV4_MOST, which f16 has no room for, has the minimum NaN: all of it reads back as NaN.

constexpr float KV4_MOST = 60000.0f;

// The codes of a lane's eight values, and the scale and minimum (f16, f16) of its group of `lanes` lanes.  `there`: the lane has values.
__device__ __forceinline__ void kv4_codes(const double (&y)[8], bool there, uint32_t lane, uint32_t lanes, uint32_t (&code)[8], uint32_t *scale_min) {
  double lo = INFINITY, hi = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    odd |= there && !(fabs(y[i]) <= (double)KV4_MOST);
    lo = there && y[i] < lo ? y[i] : lo, hi = there && y[i] > hi ? y[i] : hi;
  }
#pragma unroll
  for (uint32_t d = 1; d < 8; d *= 2) {
    const double l = __shfl_xor_sync(0xFFFFFFFFu, lo, d), h = __shfl_xor_sync(0xFFFFFFFFu, hi, d);
    if (d < lanes) lo = l < lo ? l : lo, hi = h > hi ? h : hi;
  }
  const uint32_t group = (lanes == 8 ? 0xFFu : 0xFu) << (lane & ~(lanes - 1));
  odd = (__ballot_sync(0xFFFFFFFFu, odd) & group) != 0;
  const __half least = __float2half_rn((float)lo), scale = __float2half_rn(__fmul_rn((float)(hi - lo), 1.0f / 15.0f));
  const float s = __half2float(scale);
  const double unit = s > 0.0f ? (double)__frcp_rn(s) : 0.0, from = (double)__half2float(least);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    // 1.5 * 2^52 leaves the nearest whole number in the sum's low bits
    const int n = __double2loint((y[i] - from) * unit + 6755399441055744.0);
    code[i] = odd ? 0u : (uint32_t)min(max(n, 0), 15);
  }
  *scale_min = odd ? 0x7E000000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(least) << 16;
}

// Warp `chunk` of the row's warps.
template <typename IN>
__device__ void kv4_append(const KvParams &p, uint32_t row, uint32_t chunk, double2 *turns) {
  const AttnLayer &a = p.a;
  const Kv4Shape &f = a.kv4;
  const uint32_t lane = threadIdx.x, D = a.head_dim, half = a.rope_dims / 2;
  const uint32_t sub = lane & (p.kv4_lanes - 1), heads = 32 / p.kv4_lanes, of = lane / p.kv4_lanes;
  const uint32_t d0 = sub * 8, steps = 2 * p.kv4_steps, first = chunk * p.kv4_each, end = min(steps, first + p.kv4_each);
  const bool there = d0 < D, stored = sub < 4 * f.units;
  // what value d0 + i of a key rotates with: its number, or its own
  auto mate = [&](uint32_t v) { return v >= a.rope_dims ? v : a.rope_pairs ? v ^ 1 : v < half ? v + half : v - half; };
  Raw<IN, 8> own[2], other[2];  // of two steps
  auto ask = [&](uint32_t i, Raw<IN, 8> &x, Raw<IN, 8> &y) {
    const bool key = i < p.kv4_steps;
    const uint32_t head = (key ? i : i - p.kv4_steps) * heads + of;
    x.clear(), y.clear();
    if (i >= end || head >= a.kv_heads || !there) return;
    const IN *src = key ? (const IN *)p.r.k + row * p.r.k_stride + head * D : (const IN *)p.r.v + row * p.r.v_stride + head * D;
    if (p.kv4_vec) {
      x.load(src + d0);
      if (key && !a.rope_pairs && d0 < a.rope_dims) y.load(src + mate(d0));
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x.t[e] = src[d0 + e];
      if (key && !a.rope_pairs) {
#pragma unroll
        for (int e = 0; e < 8; e++) y.t[e] = src[mate(d0 + e)];
      }
    }
  };
  grid_dep_wait();
  grid_dep_launch();
  ask(first, own[0], other[0]);
  RowPlace at;
  if (!find_row(p.kv, a.page_tokens, row, lane, &at)) return;
  if (at.pos == 0xFFFFFFFFu) {
    if (lane == 0) atomicOr(p.status, MER_DEVSTAT_BAD_CACHE);
    return;
  }
  double cw[8], sw[8];  // value i of a key: x[i] * cw[i] + its mate * sw[i], times the norm's factor
  if (first < p.kv4_steps) {
    for (uint32_t j = lane; j < half; j += 32) {
      const double x = (double)at.pos * __ldg(a.turns + j);
      double sin, cos;
      sincospi(x - 2.0 * rint(0.5 * x), &sin, &cos);
      turns[j] = make_double2(cos * (double)a.rope_scale, sin * (double)a.rope_scale);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t v = d0 + i;
      cw[i] = 1.0, sw[i] = 0.0;
      if (v < a.rope_dims) {
        const double2 t = turns[a.rope_pairs ? v / 2 : v < half ? v : v - half];
        cw[i] = t.x, sw[i] = (a.rope_pairs ? v % 2 == 0 : v < half) ? -t.y : t.y;
      }
      if (a.k_norm && there) cw[i] *= (double)__ldg(a.k_norm + v), sw[i] *= (double)__ldg(a.k_norm + mate(v));
    }
  }
  auto process = [&](uint32_t i, const Raw<IN, 8> &mine, const Raw<IN, 8> &theirs) {
    const bool key = i < p.kv4_steps;
    const uint32_t head = (key ? i : i - p.kv4_steps) * heads + of;
    float x[8];
    double y[8];
    mine.get(x);
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = (double)x[e];
    if (key) {
      double unit = 1.0;
      if (a.k_norm) {
        double sq = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) sq = fma(y[e], y[e], sq);
#pragma unroll
        for (uint32_t d = 1; d < 32; d *= 2) {
          const double o = __shfl_xor_sync(0xFFFFFFFFu, sq, d);
          sq += d < p.kv4_lanes ? o : 0.0;
        }
        unit = 1.0 / sqrt(sq / (double)D + (double)a.norm_eps);
      }
      float o[8];
      theirs.get(o);
      double z[8];
#pragma unroll
      for (int e = 0; e < 8; e++) z[e] = unit * fma(a.rope_pairs ? y[e ^ 1] : (double)o[e], sw[e], y[e] * cw[e]);
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = z[e];
    }
    uint32_t code[8], scale_min;
    const uint32_t lanes = f.group / 8;
    kv4_codes(y, there, lane, lanes, code, &scale_min);
    if (!there) {
      scale_min = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) code[e] = 0;
    }
    const uint32_t u = sub / 4, j = sub % 4, U = f.units;
    uint8_t *block = (uint8_t *)(key ? p.kv.k_pages : p.kv.v_pages) + at.page * p.kv.page_stride + head * p.kv.head_stride;
    uint8_t *codes = block + (uint64_t)at.in_page * f.token_bytes(), *scales = block + f.codes + (uint64_t)at.in_page * f.scale_bytes();
    const bool write = stored && head < a.kv_heads;
    if (key) {
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) w |= code[e] << (e / 2 * 4 + e % 2 * 16);
      if (write) *reinterpret_cast<uint32_t *>(codes + (j * U + u) * 4) = w;
    } else {
      const uint32_t w0 = code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12, w1 = code[4] | code[5] << 4 | code[6] << 8 | code[7] << 12;
      // words of unit u and the next one lie side by side: the lanes that have both exchange one of theirs
      const uint32_t r = 2 * j, given = __shfl_xor_sync(0xFFFFFFFFu, u % 2 ? w0 : w1, 4);
      if (U % 2 == 0) {
        if (write) *reinterpret_cast<uint32_t *>(codes + ((r + u % 2) * U + (u & ~1u)) * 2) = u % 2 ? given | w1 << 16 : w0 | given << 16;
      } else if (write) {
        *reinterpret_cast<uint16_t *>(codes + (r * U + u) * 2) = (uint16_t)w0;
        *reinterpret_cast<uint16_t *>(codes + ((r + 1) * U + u) * 2) = (uint16_t)w1;
      }
    }
    if (write && sub % lanes == 0) *reinterpret_cast<uint32_t *>(scales + sub / lanes * 4) = scale_min;
  };
  for (uint32_t i = first; i < end; i += 2) {
    ask(i + 1, own[1], other[1]);
    process(i, own[0], other[0]);
    ask(i + 2, own[0], other[0]);
    if (i + 1 < end) process(i + 1, own[1], other[1]);
  }
}
