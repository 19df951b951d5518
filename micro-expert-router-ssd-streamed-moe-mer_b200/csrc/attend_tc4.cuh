// The copying warps of attend_tc.cuh over a cache of 4 bits: queries as f16 rows, keys and values unpacked into f16 rows.  Included by it.
//
// The keys or the values of a block are some parts of 32 tokens (16 of wide heads), which the unpacking warps take in turn: the four that copy otherwise and the two beside the MMA
// warp, which a 16-bit cache leaves idle.  What bounds it: their unpacking, a latency of its own for every part.  2048 rows behind 8200, 32 and 4 heads of 128, captured: with four, five
// and six warps 370, 348 and 322 us; three stages of numbers instead of four 379, with one part of codes more in front 380.  A block takes 4400 cycles, 3500 from 16 bits; there are no
// registers for more warps beside the softmax's.
// Codes and scales are asked for some parts ahead (cp.async, into shared memory that one warp alone uses: no barrier but the warp's own), then a lane takes
// a token of the part, or half of one, and stores its numbers as the tiled copies of a 16-bit cache would have them.

// 4, 8 or 16 bytes, or zeros.
template <int N>
__device__ __forceinline__ void copy_some(uint32_t dst, const void *src, bool in) {
  if constexpr (N == 16)
    copy16(dst, src, in ? 16 : 0);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(in ? N : 0) : "memory");
}
// WORDS words of a token, shared out to its HALVES lanes, in vectors as wide as their addresses allow.
template <int WORDS, int HALVES>
__device__ __forceinline__ void copy_scales(uint32_t dst, const char *src, uint32_t half, bool in) {
  constexpr int N = WORDS % 4 == 0 ? 16 : WORDS % 2 == 0 ? 8 : 4;
#pragma unroll
  for (int b = 0; b < WORDS * 4; b += N)
    if (HALVES == 1 || b / N % 2 == (int)half) copy_some<N>(dst + b, in ? src + b : src, in);
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4 &v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// N 32-bit words from an address on a multiple of 4 N (at most 16) bytes.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[N]) {
  constexpr int V = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;
#pragma unroll
  for (int i = 0; i < N; i += V) {
    if constexpr (V == 4) {
      const uint4 v = lds128(a + i * 4);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    } else if constexpr (V == 2) {
      const uint2 v = lds64(a + i * 4);
      w[i] = v.x, w[i + 1] = v.y;
    } else {
      w[i] = lds32(a + i * 4);
    }
  }
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

// The numbers of a lane's words of codes into a row of keys or values.  raw: the token's bytes; dst: its row of the stage, on 128 bytes
// (its place in the swizzle is the row's low bits, exclusive-or that of the piece).  A lane has PER pieces of U words (one j of a key, a pair of r of a value).  For heads of up to 128 values a
// loop, and one for keys and values: the softmax beside it needs the instruction cache (2048 rows behind 8200: 359 us unrolled and one for each; 327 as one, 322 so, 326 not
// unrolled at all).  With wider heads the softmax waits for the unpacking, which is faster unrolled (1000 rows of 256 values behind 4000: 198, 203 to 207 so).
template <int DP, int U>
__device__ __forceinline__ void tc4_unpack(uint32_t raw, uint32_t half, uint32_t dst, uint32_t row, uint32_t wide, bool keys) {
  using S = TcShape<DP, U>;
  constexpr uint32_t PER = 4 / S::HALVES;
  uint32_t scales[(U + 3) / 4 * 4];
  auto load_scales = [&] {
#pragma unroll
    for (uint32_t i = 0; i < (U + 3) / 4; i++) {
      const uint4 v = lds128(raw + 16 * U + i * 16);
      scales[4 * i] = v.x, scales[4 * i + 1] = v.y, scales[4 * i + 2] = v.z, scales[4 * i + 3] = v.w;
    }
  };
  // Word u of a value from those of its piece: two words of 16 bits.
  auto of_value = [](const uint32_t(&w)[U], uint32_t u) { return __byte_perm(w[u / 2], w[(U + u) / 2], (u % 2 ? 0x32u : 0x10u) | ((U + u) % 2 ? 0x7600u : 0x5400u)); };
  const uint32_t to = (dst | ((row & 7) << 4)) ^ (half * (PER << 4));
  auto store = [&](uint32_t i, uint32_t u, uint32_t word) {
    const __half2 h = as_half2(wide ? scales[u / 2] : scales[u]);
    sts128((to ^ ((4 * (u & 1)) << 4) ^ (i << 4)) + (u / 2) * (TC_KB * 128), kv4_numbers(word, __low2half2(h), __high2half2(h)));
  };
  const uint32_t own = raw + half * (8 * U);
  if constexpr (S::HALVES == 1) {
    load_scales();
#pragma unroll 2
    for (uint32_t i = 0; i < PER; i++) {
      uint32_t w[U], words[U];
      lds_words<U>(own + i * (4 * U), w);
#pragma unroll
      for (uint32_t u = 0; u < U; u++) words[u] = w[u];
      if (!keys) {
#pragma unroll
        for (uint32_t u = 0; u < U; u++) words[u] = of_value(w, u);
      }
#pragma unroll
      for (uint32_t u = 0; u < U; u++) store(i, u, words[u]);
    }
  } else {
    uint32_t w[PER][U];
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) lds_words<U>(own + i * (4 * U), w[i]);
    load_scales();
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
#pragma unroll
      for (uint32_t i = 0; i < PER; i++) store(i, u, keys ? w[i][u] : of_value(w[i], u));
  }
}

template <typename IO, int DP, int U, typename Next, typename Done, typename Wait>
__device__ __forceinline__ void tc4_copies(const TcParams &p, TcControl4 &ctl, uint32_t w, uint32_t lane, uint32_t s_q, uint32_t s_ring, uint32_t s_raw, const uint32_t &turn, uint32_t *bad,
                                           const Next &next_tile, const Done &done_with, const Wait &wait) {
  using S = TcShape<DP, U>;
  constexpr uint32_t HALVES = S::HALVES, ROWS = S::RAW_ROWS, RAW = S::RAW, PARTS = TC_KB / ROWS;  // parts of a block's keys, and of its values
  const Kv4Shape &f = p.a.kv4;
  const uint32_t window = p.a.window, raw = s_raw + w * (RAW * S::RAW_STEP), wide = f.group == 64, own = lane % ROWS;
  const bool whole = p.a.page_tokens % 16 == 0;  // 16 tokens lie side by side
  uint32_t tiles = 0, halves = 0;                // halves of blocks before the tile's: half h is in stage h % STAGES
  // columns that no unit has are zeros for good: queries are zero there, but a product with what shared memory held may not be
  if constexpr (U * 32 < DP) {
    if (w < TC_LOADERS) {
      for (uint32_t i = 0; i < S::STAGES; i++)
        for (uint32_t c = 4 * U; c < DP / 8; c++)
          sts128(s_ring + i * S::STAGE + (c / 8) * (TC_KB * 128) + (w * 32 + lane) * 128 + (((c ^ lane) & 7) << 4), make_uint4(0, 0, 0, 0));
    }
  }
  while (next_tile()) {
    const TileWork t = ctl.tile[turn & 1];
    done_with();
    if (w < TC_LOADERS) {
      if (!wait(&ctl.q_empty, (tiles & 1) ^ 1)) break;
      tc4_queries<IO, DP, U>(p, t, ctl.unit[tiles & 1], w, lane, s_q);
      mbar_arrive(&ctl.q_full);
    }
    tiles++;
    const uint32_t end = t.past + t.token0 + t.tokens, start = first_seen(t, window);
    const uint32_t *const table = p.kv.page_table + (uint64_t)t.seq * p.kv.table_stride;
    const uint64_t head_at = t.kv_head * p.kv.head_stride;
    // The warp's parts are n = w, w + UNPACKERS, ..: part n % PARTS of the keys or the values (n / PARTS even or odd) of block lo + n / (2 PARTS).
    const uint32_t parts = (t.hi - t.lo) * 2 * PARTS;
    auto token_of = [&](uint32_t n) { return (t.lo + n / (2 * PARTS)) * TC_KB + n % PARTS * ROWS + own; };
    auto entry = [&](uint32_t n) {
      const uint32_t key = token_of(n), at = divided(key, p.kv.page_tokens);
      return n < parts && key >= start && key < end && at < p.kv.table_stride ? table[at] : 0xFFFFFFFFu;
    };
    uint32_t number = entry(w), slot = 0;  // of the next part that is asked for
    auto ask = [&](uint32_t n) {
      if (n < parts) {
        const uint32_t key = token_of(n);
        const bool seen = key >= start && key < end, there = seen && number < p.kv.n_pages;
        if (seen && !there) *bad = 1;
        const uint32_t in_page = key - divided(key, p.kv.page_tokens) * p.a.page_tokens;
        const uint64_t block = there ? number * p.kv.page_stride + head_at : 0;
        const uint64_t codes = block + in_page * (16 * U);
        number = entry(n + S::UNPACKERS);
        const char *const base = (const char *)(n / PARTS % 2 ? p.kv.v_pages : p.kv.k_pages);
        const uint32_t dst = raw + slot * S::RAW_STEP;
        const uint32_t all = __ballot_sync(0xFFFFFFFFu, there);
        if (whole && all == 0xFFFFFFFFu) {
          const uint64_t run0 = __shfl_sync(0xFFFFFFFFu, codes, 0), run1 = HALVES == 1 ? __shfl_sync(0xFFFFFFFFu, codes, 16) : run0;
#pragma unroll
          for (uint32_t i = 0; i < U * ROWS / 32; i++) {
            const uint32_t e = i * 32 + lane, r = e / U, c = e - r * U;
            copy16(dst + r * S::RAW_STRIDE + c * 16, base + (HALVES == 1 && (U % 2 ? e >= 16 * U : i >= U / 2) ? run1 + (e - 16 * U) * 16 : run0 + e * 16), 16);
          }
        } else {
#pragma unroll
          for (uint32_t i = 0; i < U * ROWS / 32; i++) {
            const uint32_t e = i * 32 + lane, r = e / U, c = e - r * U;
            const uint64_t at = __shfl_sync(0xFFFFFFFFu, codes, r);
            const bool in = all >> r & 1;
            copy16(dst + r * S::RAW_STRIDE + c * 16, in ? base + at + c * 16 : base, in ? 16 : 0);
          }
        }
        const char *const from = there ? base + block + f.codes + in_page * f.scale_bytes() : base;
        const uint32_t to = dst + own * S::RAW_STRIDE + 16 * U;
        if (wide)
          copy_scales<(U + 1) / 2, HALVES>(to, from, lane / ROWS, there);
        else
          copy_scales<U, HALVES>(to, from, lane / ROWS, there);
      }
      slot = slot + 1 == RAW ? 0 : slot + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (uint32_t i = 0; i < RAW - 1; i++) ask(w + i * S::UNPACKERS);
    uint32_t taken = 0;
    bool ok = true;
    for (uint32_t n = w; n < parts; n += S::UNPACKERS) {
      ask(n + (RAW - 1) * S::UNPACKERS);
      copies_left<RAW - 1>();
      __syncwarp();
      const uint32_t h = halves + n / PARTS, stage = h % S::STAGES, row = n % PARTS * ROWS + own;
      if (!(ok = wait(&ctl.empty[stage], (h / S::STAGES & 1) ^ 1))) break;
      const uint32_t from = raw + taken * S::RAW_STEP + own * S::RAW_STRIDE, dst = s_ring + stage * S::STAGE + row * 128;
      const bool keys = n / PARTS % 2 == 0;
      if constexpr (HALVES == 1)
        tc4_unpack<DP, U>(from, lane / ROWS, dst, row, wide, keys);
      else if (keys)
        tc4_unpack<DP, U>(from, lane / ROWS, dst, row, wide, true);
      else
        tc4_unpack<DP, U>(from, lane / ROWS, dst, row, wide, false);
      taken = taken + 1 == RAW ? 0 : taken + 1;
      // The MMA warp makes the stage visible to the tensor core.
      mbar_arrive(&ctl.full[stage]);
      __syncwarp();  // the part's place may be asked for again
    }
    if (!ok) break;
    halves += (t.hi - t.lo) * 2;
  }
}
