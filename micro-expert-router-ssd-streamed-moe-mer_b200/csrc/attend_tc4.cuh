// The copying warps of attend_tc.cuh over a cache of 4 bits: queries as f16 rows, keys and values unpacked into f16 rows.  Included by it.
//
// Codes and scales are asked for some steps ahead (cp.async, into a part of shared memory that one warp alone uses: no barrier but the warp's own), then a lane takes
// a token of the step, or half of one, and stores its numbers as the tiled copies of a 16-bit cache would have them.

// 4, 8 or 16 bytes, or zeros.
template <int N>
__device__ __forceinline__ void copy_some(uint32_t dst, const void *src, bool in) {
  if constexpr (N == 16)
    copy16(dst, src, in ? 16 : 0);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(in ? N : 0) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4 &v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Queries of a tile as f16: a row is divided by a power of two that brings its largest value between 1 and 2, which f16 holds as exactly as its own type did down to 2^-14
// of that; the power goes to the scores' factor.
template <typename IO, int DP, int U>
__device__ __forceinline__ void tc4_queries(const TcParams &p, const TileWork &t, float *unit, uint32_t w, uint32_t lane, uint32_t s_q) {
  using S = TcShape<DP, U>;
  constexpr uint32_t PIECES = DP / 8, AT_ONCE = 32 / PIECES, ROWS = S::R / TC_LOADERS;
  const uint32_t c = lane % PIECES, rows = t.tokens * t.heads, D = p.a.head_dim;
#pragma unroll 4
  for (uint32_t i = 0; i < ROWS; i += AT_ONCE) {
    const uint32_t r = w * ROWS + i + lane / PIECES, tok = r / t.heads;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (r < rows && c * 8 < D)
      raw = *reinterpret_cast<const uint4 *>((const IO *)p.q + (uint64_t)(t.row0 + t.token0 + tok) * p.q_stride + (uint64_t)(t.head0 + r - tok * t.heads) * D + c * 8);
    float x[8], top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = Num<IO>::f(reinterpret_cast<const IO *>(&raw)[e]), top = fmaxf(top, fabsf(x[e]));
#pragma unroll
    for (uint32_t d = 1; d < PIECES; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
    const float per = __uint_as_float((254 - e) << 23);
    sts128(s_q + (c / 8) * S::QSUB + r * 128 + (((c ^ r) & 7) << 4),
           make_uint4(Num<__half>::pack(x[0] * per, x[1] * per), Num<__half>::pack(x[2] * per, x[3] * per), Num<__half>::pack(x[4] * per, x[5] * per), Num<__half>::pack(x[6] * per, x[7] * per)));
    if (c == 0) unit[r] = __uint_as_float(e << 23);
  }
}

// The numbers of a lane's words of codes into a row of keys or values.  raw: the token's bytes; dst: its row of the stage.
template <int DP, int U, bool KEYS>
__device__ __forceinline__ void tc4_unpack(uint32_t raw, uint32_t half, uint32_t dst, uint32_t row, uint32_t wide) {
  using S = TcShape<DP, U>;
  constexpr uint32_t PER = 4 / S::HALVES;  // fours of words (j, or pairs of r) of a lane
  static_assert(PER * U % 4 == 0, "a lane's words are whole vectors");
  uint32_t words[PER * U], scales[(U + 3) / 4 * 4];
#pragma unroll
  for (uint32_t i = 0; i < PER * U / 4; i++) {
    const uint4 v = lds128(raw + half * (8 * U) + i * 16);
    words[4 * i] = v.x, words[4 * i + 1] = v.y, words[4 * i + 2] = v.z, words[4 * i + 3] = v.w;
  }
#pragma unroll
  for (uint32_t i = 0; i < (U + 3) / 4; i++) {
    const uint4 v = lds128(raw + 16 * U + i * 16);
    scales[4 * i] = v.x, scales[4 * i + 1] = v.y, scales[4 * i + 2] = v.z, scales[4 * i + 3] = v.w;
  }
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const __half2 h = as_half2(wide ? scales[u / 2] : scales[u]);
    const __half2 scale = __low2half2(h), least = __high2half2(h);
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) {
      uint32_t word;
      if constexpr (KEYS) {
        word = words[i * U + u];
      } else {
        const uint32_t a = 2 * i * U + u, b = a + U;  // two words of 16 bits
        word = __byte_perm(words[a / 2], words[b / 2], (a % 2 ? 0x32u : 0x10u) | (b % 2 ? 0x7600u : 0x5400u));
      }
      const uint32_t col = 4 * (u & 1) + half * PER + i;
      sts128(dst + (u / 2) * (TC_KB * 128) + ((col ^ (row & 7)) << 4), kv4_numbers(word, scale, least));
    }
  }
}

template <typename IO, int DP, int U, typename Next, typename Done, typename Wait>
__device__ __forceinline__ void tc4_copies(const TcParams &p, TcControl4 &ctl, uint32_t w, uint32_t lane, uint32_t s_q, uint32_t s_ring, uint32_t s_raw, const uint32_t &turn, uint32_t *bad,
                                           const Next &next_tile, const Done &done_with, const Wait &wait) {
  using S = TcShape<DP, U>;
  constexpr uint32_t HALVES = S::HALVES, ROWS = S::RAW_ROWS, RAW = S::RAW;
  const Kv4Shape &f = p.a.kv4;
  const uint32_t window = p.a.window, raw = s_raw + w * (RAW * S::RAW_STEP), wide = f.group == 64;
  uint32_t stage = 0, phase = 0, tiles = 0;
  // columns that no unit has are zeros for good: queries are zero there, but a product with what shared memory held may not be
  if constexpr (U * 32 < DP) {
    for (uint32_t i = 0; i < S::STAGES; i++)
      for (uint32_t c = 4 * U; c < DP / 8; c++)
        sts128(s_ring + i * S::STAGE + (c / 8) * (TC_KB * 128) + (w * 32 + lane) * 128 + (((c ^ lane) & 7) << 4), make_uint4(0, 0, 0, 0));
  }
  while (next_tile()) {
    const TileWork t = ctl.tile[turn & 1];
    done_with();
    if (!wait(&ctl.q_empty, (tiles & 1) ^ 1)) break;
    tc4_queries<IO, DP, U>(p, t, ctl.unit[tiles & 1], w, lane, s_q);
    proxy_fence();
    mbar_arrive(&ctl.q_full);
    tiles++;
    const uint32_t end = t.past + t.token0 + t.tokens, start = first_seen(t, window);
    const uint32_t *const table = p.kv.page_table + (uint64_t)t.seq * p.kv.table_stride;
    auto entry = [&](uint32_t blk) {
      const uint32_t key = blk * TC_KB + w * 32 + lane, slot = divided(key, p.kv.page_tokens);
      return blk < t.hi && key >= start && key < end && slot < p.kv.table_stride ? table[slot] : 0xFFFFFFFFu;
    };
    // Step n is of block lo + n / (2 HALVES): keys, then values, each in HALVES parts of the warp's tokens.
    const uint32_t steps = (t.hi - t.lo) * 2 * HALVES;
    uint32_t number = entry(t.lo), in_page = 0, slot = 0;  // slot: of the next step that is asked for
    uint64_t block = 0;                                    // where the lane's token's page begins
    auto ask = [&](uint32_t n) {
      if (n < steps) {
        if (n % (2 * HALVES) == 0) {
          const uint32_t blk = t.lo + n / (2 * HALVES), key = blk * TC_KB + w * 32 + lane;
          const bool seen = key >= start && key < end, there = seen && number < p.kv.n_pages;
          if (seen && !there) *bad = 1;
          in_page = there ? key - divided(key, p.kv.page_tokens) * p.a.page_tokens : 0xFFFFFFFFu;
          block = there ? number * p.kv.page_stride + t.kv_head * p.kv.head_stride : 0;
          number = entry(blk + 1);
        }
        const char *const base = (const char *)(n / HALVES % 2 ? p.kv.v_pages : p.kv.k_pages);
        const uint32_t first = n % HALVES * ROWS, dst = raw + slot * S::RAW_STEP;
#pragma unroll
        for (uint32_t i = 0; i < U * ROWS / 32; i++) {
          const uint32_t e = i * 32 + lane, r = e / U, c = e - r * U;
          const uint64_t at = __shfl_sync(0xFFFFFFFFu, block, first + r);
          const uint32_t in = __shfl_sync(0xFFFFFFFFu, in_page, first + r);
          const bool there = in != 0xFFFFFFFFu;
          copy_some<16>(dst + r * S::RAW_STRIDE + c * 16, there ? base + at + (uint64_t)in * (16 * U) + c * 16 : base, there);
        }
        const uint32_t r = lane % ROWS, c = lane / ROWS;
        const uint64_t at = __shfl_sync(0xFFFFFFFFu, block, first + r);
        const uint32_t in = __shfl_sync(0xFFFFFFFFu, in_page, first + r), bytes = f.scale_bytes();
        const bool there = in != 0xFFFFFFFFu;
        const char *const from = there ? base + at + f.codes + (uint64_t)in * bytes : base;
        const uint32_t to = dst + r * S::RAW_STRIDE + 16 * U;
        if (bytes % 16 == 0) {
          for (uint32_t b = c * 16; b < bytes; b += HALVES * 16) copy_some<16>(to + b, there ? from + b : base, there);
        } else if (bytes % 8 == 0) {
          for (uint32_t b = c * 8; b < bytes; b += HALVES * 8) copy_some<8>(to + b, there ? from + b : base, there);
        } else {
          for (uint32_t b = c * 4; b < bytes; b += HALVES * 4) copy_some<4>(to + b, there ? from + b : base, there);
        }
      }
      slot = slot + 1 == RAW ? 0 : slot + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (uint32_t n = 0; n < RAW - 1; n++) ask(n);
    uint32_t taken = 0;
    bool ok = true;
    for (uint32_t n = 0; n < steps; n++) {
      ask(n + RAW - 1);
      copies_left<RAW - 1>();
      __syncwarp();
      if (n % HALVES == 0 && !(ok = wait(&ctl.empty[stage], phase ^ 1))) break;
      const uint32_t r = lane % ROWS, half = lane / ROWS, row = w * 32 + n % HALVES * ROWS + r;
      const uint32_t from = raw + taken * S::RAW_STEP + r * S::RAW_STRIDE, dst = s_ring + stage * S::STAGE + row * 128;
      if (n / HALVES % 2)
        tc4_unpack<DP, U, false>(from, half, dst, row, wide);
      else
        tc4_unpack<DP, U, true>(from, half, dst, row, wide);
      taken = taken + 1 == RAW ? 0 : taken + 1;
      if (n % HALVES == HALVES - 1) {
        proxy_fence();
        mbar_arrive(&ctl.full[stage]);
        stage = stage + 1 == S::STAGES ? 0 : stage + 1, phase ^= stage == 0;
      }
      __syncwarp();  // the step's place may be asked for again
    }
    if (!ok) break;
  }
}
