// A tile: included in kernels of T, D, PAGED, Q8 and PREFIX that have a (FwdArgs), smem
// (tile_bytes<D, Q8>() of LDS), s_bad and s_skip[4] (LDS), and the tile's block of blocks; it
// returns from them.  (As a function it compiles to code that is 6 % slower over pages.)
//
// The loop is software-pipelined by halves of 32 keys: while a half's probabilities are
// formed in the VALU, the matrix cores form the next half's scores, then its product with V
// while the second sixteen probabilities and the next half's maximum are formed.  A step of
// the loop multiplies K's keys 64 j .. 64 j + 63 and V's 64 j - 32 .. 64 j + 31, so both
// tiles have two buffers, and arrive in LDS directly, a step ahead of their use.
// Workgroups of a compute unit: two at head size 128, for the registers; at 64 three, which
// hides more of the exponentials (404 -> 396 us on packed prompts).  Outside the loop registers
// spill: 50 at 128 and 38 at 64 over contiguous keys, 4 and 6 over pages.
//
// Q8: a cache of 8 bits.  Its rows arrive in LDS as they are, in the upper halves of the places
// that a wave's 16 rows of either tile will take, and the wave turns them into the inputs' type
// there before the step that reads them, so the rest is the same.
// PREFIX: the rows of all sequences behind one prefix attend all its keys, and leave their
// shares.
  typedef typename El<T>::v8 v8;
  constexpr int NC = D / 8;                 // 16-byte chunks of a row
  constexpr int RI = 64 / NC, NL = 16 / RI; // rows of a wave's load, loads of its 16 rows of a tile
  constexpr int NS = D / 16, ND = D / 32;
  constexpr int TILE = BN * D * 2;          // bytes
  // K, K, V, V; of 8 bits two steps' scales too, a wave's 16 rows of either tile in 32 words
  constexpr int SCALES = 4 * TILE;

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // uniform, and known to be
  const int kvh = block % a.HKV;
  const Tile t = next_tile<BM, true>(a.seqs, PAGED ? a.pages.lens : nullptr, place(block / a.HKV, blocks / a.HKV, a.places), a.slots,
                                       a.split);
  if (t.row0 >= t.rows || t.row0 < 0) return;

  const int row = t.row0 + wave * 32 + l32;
  const int rowc = min(row, t.rows - 1);
  const int tok = fdiv(rowc, a.G), head = kvh * a.G.d + rowc - tok * a.G.d;
  if (PREFIX && t.seq < 0) {                // rows behind no prefix
    if (row < t.rows && h == 0)
      share_stats<D>(a, 0, (int64_t)(t.bos + tok) * a.H + head)[0] = __builtin_bit_cast(float, NO_SHARE);
    return;
  }
  if (t.seq < 0) {                          // rows of no sequence
    if (a.fill && row < t.rows) {
      char* orow = a.o + (int64_t)(t.bos + tok) * a.o_ts + (int64_t)head * a.o_hs;
#pragma unroll
      for (int i = 0; i < NS; ++i) *reinterpret_cast<u32x4*>(orow + 32 * i + 16 * h) = u32x4{0, 0, 0, 0};
      if (a.lse && h == 0) a.lse[(int64_t)(t.bos + tok) * a.H + head] = NEG_INF;
    }
    return;
  }

  int keys = t.tokens;
  if constexpr (PAGED)
    keys = (int)min((int64_t)max(uniform_load(a.pages.lens, t.seq), 0),
                    (int64_t)a.pages.width * a.pages.page.d);
  keys = __builtin_amdgcn_readfirstlane(keys);
  // token i attends keys 0 .. off + i; behind a prefix each attends all
  const int off = PREFIX ? keys - 1 : keys - t.tokens;
  auto token_of = [&](int r) __attribute__((always_inline)) { return PREFIX ? 0 : fdiv(r, a.G); };
  const int klast = PREFIX ? off : off + tok;
  const int wrow = t.row0 + wave * 32;
  const int w_first = off + token_of(min(wrow, t.rows - 1));             // least last key of the wave's rows
  const int w_last = off + token_of(min(wrow + 31, t.rows - 1));         // and greatest
  const int wg_first = off + token_of(t.row0);
  const int wg_last = off + token_of(min(t.row0 + BM, t.rows) - 1);
  const int nt_all = wg_last < 0 ? 0 : wg_last / BN + 1;
  const int sp = t.sp, ns = t.ns;
  const int j_beg = (int)((int64_t)nt_all * sp / ns), j_end = (int)((int64_t)nt_all * (sp + 1) / ns);
  const int u_beg = 2 * j_beg, u_last = min(2 * j_end - 1, w_last < 0 ? -1 : w_last / 32);   // the wave's halves
  if (tid < 4) s_skip[tid] = -1;
  if (tid == 0) s_bad = 0;

  v8 qf[NS];
  {
    const char* qp = a.q + (int64_t)(t.bos + tok) * a.q_ts + (int64_t)head * a.q_hs + 16 * h;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const v8*>(qp + 32 * s);
  }

  // Staging: the wave brings rows 16 wave .. 16 wave + 15 of a tile, RI to a load; the lane's
  // chunk is the one that the swizzle puts at its place.
  uint32_t koff[NL], voff[NL];
  const int64_t kts = PAGED ? a.pages.k_ts : a.k_ts, vts = PAGED ? a.pages.v_ts : a.v_ts;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = i * RI + lane / NC, c = swz<D>(wave * 16 + r, lane % NC);
    koff[i] = (uint32_t)(r * (int)kts + 16 * c);
    voff[i] = (uint32_t)(r * (int)vts + 16 * c);
  }
  const char* kbase = (PAGED ? a.pages.k : a.k + (int64_t)t.bos * a.k_ts) + (int64_t)kvh * (PAGED ? a.pages.k_hs : a.k_hs);
  const char* vbase = (PAGED ? a.pages.v : a.v + (int64_t)t.bos * a.v_ts) + (int64_t)kvh * (PAGED ? a.pages.v_hs : a.v_hs);
  const bool whole = !PAGED || a.pages.page.d % 16 == 0;   // the wave's 16 rows lie in one page
  // s_skip[j & 3] = j + 1 (-1 at first): some page of key tile j lies outside the cache.  Only
  // the staging of the tile's keys says so, in the step before the tile's own; while a step's
  // waves read the flags of tiles j and j - 1 (mend has a barrier behind them), stage(j + 1)
  // writes tile j + 1's alone.  Values need none: those that a product takes are of tiles whose
  // keys were staged.
  auto stage_rows = [&](int j, int r0, bool value) __attribute__((always_inline)) {
    const uint32_t lds = lds_addr(smem) + (value ? 2 * TILE : 0) + ((j - j_beg) & 1) * TILE + wave * 16 * D * 2;
    const char* base = value ? vbase : kbase;
    const int64_t ts = value ? vts : kts;
    if (!PAGED && r0 >= 0 && r0 + 16 <= keys) {
      const char* b = uniform_ptr(base + r0 * ts);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(lds + i * RI * D * 2, b, value ? voff[i] : koff[i]);
    } else if (PAGED && whole) {
      // rows behind the last key are the page's own: what they hold is masked
      const int r = max(min(r0, (keys - 1) & ~15), 0), p = fdiv(r, a.pages.page);
      int id = uniform_load(a.pages.table, t.seq * a.pages.table_stride + __builtin_amdgcn_readfirstlane(p));
      if ((unsigned)id >= (unsigned)a.pages.num_pages) {
        if (!value && r0 < keys) s_skip[j & 3] = j + 1;
        id = 0;
      }
      const char* b = uniform_ptr(base + id * (value ? a.pages.v_ps : a.pages.k_ps) + (r - p * a.pages.page.d) * ts);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(lds + i * RI * D * 2, b, value ? voff[i] : koff[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int q = r0 + i * RI + lane / NC, r = max(min(q, keys - 1), 0);
        const char* b = base;
        if constexpr (PAGED) {
          const int p = fdiv(r, a.pages.page);
          int id = a.pages.table[t.seq * a.pages.table_stride + p];
          if ((unsigned)id >= (unsigned)a.pages.num_pages) {
            if (!value && q < keys) s_skip[j & 3] = j + 1;
            id = 0;
          }
          b += id * (value ? a.pages.v_ps : a.pages.k_ps) + (r - p * a.pages.page.d) * ts;
        } else {
          b += r * ts;
        }
        dma16(lds + i * RI * D * 2, b + 16 * swz<D>(wave * 16 + i * RI + lane / NC, lane % NC));
      }
    }
  };
  // Of a cache of 8 bits: the wave's rows of step j's tiles as they are, RI8 to a load, and
  // their bytes of scale, a word each (lanes 0 .. 15 keys, 16 .. 31 values); vlive, a bit for
  // each of the values' rows that is a key.
  constexpr int RI8 = 1024 / D, NL8 = 16 / RI8;
  uint32_t vlive = 0;
  auto stage_rows8 = [&](int j, bool value, const uint8_t*& sc) __attribute__((always_inline)) {
    const int r0 = j * BN - (value ? 32 : 0) + wave * 16;
    const uint32_t lds = lds_addr(smem) + (value ? 2 * TILE : 0) + ((j - j_beg) & 1) * TILE + wave * 16 * D * 2 + 16 * D;
    const char* base = value ? vbase : kbase;
    const int64_t ps = value ? a.pages.v_ps : a.pages.k_ps, ts = value ? vts : kts;
    const uint8_t* sbase = value ? a.pages.v_sc + kvh * a.pages.v_sc_hs : a.pages.k_sc + kvh * a.pages.k_sc_hs;
    const int64_t sps = value ? a.pages.v_sc_ps : a.pages.k_sc_ps;
    const bool mine = value == (bool)((lane >> 4) & 1);
    uint32_t live = r0 < 0 ? 0 : (1u << min(max(keys - r0, 0), 16)) - 1;   // r0 is a multiple of 16
    if (whole) {
      const int r = max(min(r0, (keys - 1) & ~15), 0), p = fdiv(r, a.pages.page);
      int id = uniform_load(a.pages.table, t.seq * a.pages.table_stride + __builtin_amdgcn_readfirstlane(p));
      if ((unsigned)id >= (unsigned)a.pages.num_pages) {
        if (!value && live) s_skip[j & 3] = j + 1;
        id = 0;
        live = 0;
      }
      const int in = r - p * a.pages.page.d;
      const char* b = uniform_ptr(base + id * ps + in * ts);
#pragma unroll
      for (int i = 0; i < NL8; ++i)
        dma16(lds + i * 1024, b, (uint32_t)((i * RI8 + lane / (D / 16)) * (int)ts + 16 * (lane % (D / 16))));
      if (mine) sc = sbase + id * sps + in + (lane & 15);
    } else {
      int in;
      auto page_of = [&](int x) __attribute__((always_inline)) {   // of row x, -1 outside the cache, and its place
        const int r = max(min(r0 + x, keys - 1), 0), p = fdiv(r, a.pages.page);
        const int id = a.pages.table[t.seq * a.pages.table_stride + p];
        in = r - p * a.pages.page.d;
        return (unsigned)id < (unsigned)a.pages.num_pages ? id : -1;
      };
      const int id = page_of(lane & 15);
      const uint32_t there = (uint32_t)__ballot(id >= 0) & 0xffffu;
      if (!value && (live & ~there)) s_skip[j & 3] = j + 1;
      live &= there;
      if (mine) sc = sbase + max(id, 0) * sps + in;
#pragma unroll
      for (int i = 0; i < NL8; ++i) {
        const int64_t page = max(page_of(i * RI8 + lane / (D / 16)), 0);
        dma16(lds + i * 1024, base + page * ps + in * ts + 16 * (lane % (D / 16)));
      }
    }
    return live;
  };
  auto stage8 = [&](int j) __attribute__((always_inline)) {
    const uint8_t* sc = a.pages.k_sc + kvh * a.pages.k_sc_hs;   // any byte, where the step brings no keys
    if (j < j_end) stage_rows8(j, false, sc);
    vlive = stage_rows8(j, true, sc);
    dma1(lds_addr(smem) + SCALES + ((j - j_beg) & 1) * 1024 + wave * 256, sc);
  };
  auto stage = [&](int j) __attribute__((always_inline)) {                 // the keys and values of step j
    if constexpr (Q8) {
      stage8(j);
    } else {
      if (j < j_end) stage_rows(j, j * BN + wave * 16, false);
      stage_rows(j, j * BN - 32 + wave * 16, true);
    }
  };
  // The wave's rows of step j's tiles in the inputs' type, where they lie: all are read before
  // the first is written.  Rows of V that are no keys become 0, and values that are not finite
  // where some row's keys end among them, as in mend().
  auto widen = [&](int j) __attribute__((always_inline)) {
    constexpr int NP = D / 32;              // pieces of eight values a lane
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(smem + SCALES + ((j - j_beg) & 1) * 1024 + wave * 256);
    const bool edge = j * BN - 32 + BN > wg_first + 1;
#pragma unroll
    for (int value = 0; value < 2; ++value) {
      if (!value && j >= j_end) continue;
      char* rows = smem + (value ? 2 * TILE : 0) + ((j - j_beg) & 1) * TILE + wave * 16 * D * 2;
      u32x2 x[NP];
      uint32_t code[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        x[i] = *reinterpret_cast<const u32x2*>(rows + 16 * D + 8 * (lane + 64 * i));
        code[i] = scales[16 * value + (lane + 64 * i) / NC];
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (value && (edge || vlive != 0xffffu)) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t n = nan_bytes(x[i][z]);
            const bool key = (vlive >> ((lane + 64 * i) / NC)) & 1;
            bad |= key && edge && n;
            x[i][z] = key ? (edge ? x[i][z] & ~n : x[i][z]) : 0;
            if (!key) code[i] = 1;          // the power may be anything too
          }
        if (bad) s_bad = 1;
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = (lane + 64 * i) / NC, c = lane % NC;
        v8 y = from_e4m3<T>(x[i], scale_of(code[i]));
        if constexpr (__is_same(T, f16)) {
          if (code[i] >= 127 + 8) {         // 448 times it passes fp16's range: the largest value there, NaN as it is
#pragma unroll
            for (int z = 0; z < 8; ++z) {
              const float f = (float)y[z];
              if (f > 65504.f) y[z] = (f16)65504.f;
              if (f < -65504.f) y[z] = (f16)-65504.f;
            }
          }
        }
        *reinterpret_cast<v8*>(rows + r * D * 2 + swz<D>(wave * 16 + r, c) * 16) = y;
      }
    }
  };
  // Rows of step j's V that are no keys to 0 (their probability is 0, their memory anything).
  // Where some row's keys end among them, so do values that are not finite: 0 times one is not
  // 0, and the product would spoil the rows that do not attend it; add_nonfinite() brings them
  // to those that do.
  auto mend = [&](int j) __attribute__((always_inline)) {
    const int r0 = j * BN - 32;
    const bool edge = r0 + BN > wg_first + 1, out = r0 < j_beg * BN || r0 + BN > keys;
    const bool hole = PAGED && (s_skip[j & 3] == j + 1 || s_skip[(j - 1) & 3] == j);
    if (!(edge || out || hole)) return;
    T* Vb = reinterpret_cast<T*>(smem + (2 + ((j - j_beg) & 1)) * TILE);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < BN * NC / 256; ++i) {
      const int q = r0 + (tid + 256 * i) / NC;
      u32x4* p = reinterpret_cast<u32x4*>(Vb + (tid + 256 * i) * 8);
      bool key = q >= 0 && q < keys;
      if constexpr (PAGED) {
        if (hole && key) key = key_row<T, true>(a, t, kvh, q, true) != nullptr;
      }
      if (!key) {
        *p = u32x4{0, 0, 0, 0};
      } else if (edge && any_nonfinite<T>(*p)) {
        uint16_t* e = reinterpret_cast<uint16_t*>(p);
#pragma unroll 1
        for (int z = 0; z < 8; ++z)
          if (nonfinite<T>(e[z])) e[z] = 0;
        bad = true;
      }
    }
    if (bad) s_bad = 1;
    __syncthreads();
  };

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x16{0};
  // reference maximum of the raw scores, m c (where there is none, so low that any score makes
  // P infinite), and own half's sum of P
  float m = NEG_INF, mc = NO_MC, l = 0.f;

  // the lane's byte offsets into the tiles; flip() takes them to the other buffers
  int ko[NS], vo[ND], vu[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s) ko[s] = (l32 * D + swz<D>(l32, 2 * s + h) * 8) * 2;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    vo[d] = tr_offset<D>(lane, d, false) * 2;
    vu[d] = tr_offset<D>(lane, d, true) * 2;
  }
  auto flip = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NS; ++s) ko[s] ^= TILE;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      vo[d] ^= TILE;
      vu[d] ^= TILE;
    }
  };
  auto scores = [&](int kt, f32x16& st) __attribute__((always_inline)) {
    st = f32x16{0};
#pragma unroll
    for (int s = 0; s < NS; ++s)
      st = El<T>::mma32(*reinterpret_cast<const v8*>(smem + ko[s] + kt * 32 * D * 2), qf[s], st);
  };
  auto mask = [&](int u, f32x16& st) __attribute__((always_inline)) {
    const int k0 = u * 32 + 4 * h;
    if (u * 32 + 31 > w_first) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k0 + 8 * (i >> 2) + (i & 3) > klast) st[i] = NEG_INF;
    }
    if constexpr (PAGED) {
      if (s_skip[(u >> 1) & 3] == (u >> 1) + 1) {   // pages outside the cache hold no keys
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = k0 + 8 * (i >> 2) + (i & 3);
          if (key <= klast && !key_row<T, true>(a, t, kvh, key, false)) st[i] = NEG_INF;
        }
      }
    }
  };
  auto maximum = [&](const f32x16& st) __attribute__((always_inline)) {
    float x = fmaxf(st[0], st[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) x = fmaxf(x, st[i]);
    return half_max(x);
  };
  auto follow = [&](float mx) __attribute__((always_inline)) {   // the reference becomes the running maximum
    const float mn = fmaxf(m, mx), f = m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
    m = mn;
    mc = m == NEG_INF ? NO_MC : m * a.c;
    l *= f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] *= f;
  };
  // The reference need not be the maximum, only near it.  EAGER: it follows the maximum of the
  // next half where that is more than 2^8 ahead.  Otherwise the maxima are not formed at all:
  // P and its sum are formed with the reference at hand, and a half whose sum passes 2^12 in
  // some row (so also one with a row's first keys) is formed again after the reference has
  // followed.  P stays below 2^12 either way, inside either type, and O is seldom rescaled.
  // The second way takes 10 vector instructions less of 86 a half (prompt of 32768, 16 / 4
  // heads: 4.03 -> 3.87 ms) and 16 registers more, which the paged kernel does not have (pieces
  // of prompts 852 -> 834 us, but draft tokens 81 -> 89).
  constexpr bool EAGER = PAGED;
  auto element = [&](const f32x16& st, int i, float* p, float& sum) __attribute__((always_inline)) {
    p[i] = __builtin_amdgcn_exp2f(st[i] * a.c - mc);
    sum += p[i];
  };
  auto settle = [&](const f32x16& st, float* p, float& sum) __attribute__((always_inline)) {
    if (__any(sum > 4096.f)) {
      follow(maximum(st));
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) element(st, i, p, sum);
    }
    l += sum;
  };
  // P in the inputs' type: each is off by half a step of itself, so O by at most half a step of
  // sum p |v|, what its own rounding costs it too.  What that leaves as a product of its own, as
  // in the kernels of few rows, which wait for memory, would be half as many matrix products
  // again here, where they are the bound.
  auto pack = [&](const float* p) __attribute__((always_inline)) {
    return pack8<T>(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
  };
  // half u, whose scores are cur, against V's rows r of its tile; nxt receives the next
  // half's scores from K's half kt; the tiles are the buffers at `at`
  constexpr int AHEAD = 2;                  // LDS reads run so many products ahead
  auto half = [&](int u, const f32x16& cur, f32x16& nxt, int at, int kt, int r) __attribute__((always_inline)) {
    const char *Kb = smem + at + kt * 32 * D * 2, *Vb = smem + at + 2 * TILE + r * D * 2;
    constexpr int E = EAGER ? 8 : 16;       // elements of P formed beside the scores
    v8 kf[NS], vf[2 * ND], pf[2];
    float p[16], sum = 0.f, mx = NEG_INF;
    auto key_of = [&](int s) __attribute__((always_inline)) { kf[s] = *reinterpret_cast<const v8*>(Kb + ko[s]); };
    auto value_of = [&](int g) __attribute__((always_inline)) {
      const char* v = Vb + (g / ND) * 16 * D * 2;
      vf[g] = join<T>(tr4<T>(reinterpret_cast<const T*>(v + vo[g % ND])), tr4<T>(reinterpret_cast<const T*>(v + vu[g % ND])));
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) key_of(s);
    fence();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if (s + AHEAD < NS) key_of(s + AHEAD);
      else value_of(s + AHEAD - NS);
      nxt = El<T>::mma32(kf[s], qf[s], s == 0 ? f32x16{0} : nxt);
#pragma unroll
      for (int i = s * E / NS; i < (s + 1) * E / NS; ++i) element(cur, i, p, EAGER ? l : sum);
      fence();
    }
    if constexpr (EAGER) {
      pf[0] = pack(p);
      asm volatile("" : "+v"(pf[0]));       // formed here, not behind the mask
    } else {
      settle(cur, p, sum);
    }
    mask(u + 1, nxt);
    if constexpr (!EAGER) pf[0] = pack(p);
#pragma unroll
    for (int g = 0; g < 2 * ND; ++g) {
      if (g + AHEAD < 2 * ND) value_of(g + AHEAD);
      acc[g % ND] = El<T>::mma32(vf[g], pf[g / ND], acc[g % ND]);
      if constexpr (EAGER) {
        if (g < ND) {
#pragma unroll
          for (int i = g * 8 / ND; i < (g + 1) * 8 / ND; ++i) element(cur, 8 + i, p, l);
          if (g == ND - 1) pf[1] = pack(p + 8);
        } else {
#pragma unroll
          for (int i = (g - ND) * 16 / ND; i < (g - ND + 1) * 16 / ND; ++i) mx = fmaxf(mx, nxt[i]);
        }
      } else {
        if (g == 0) pf[1] = pack(p + 8);
      }
      fence();
    }
    if constexpr (EAGER) {
      mx = half_max(mx);
      if (__any((mx - m) * a.c > 8.f)) follow(mx);
    }
  };
  auto last_half = [&](const f32x16& cur, int r) __attribute__((always_inline)) {
    float p[16], sum = 0.f;
    if constexpr (!EAGER) {
#pragma unroll
      for (int i = 0; i < 16; ++i) element(cur, i, p, sum);
      settle(cur, p, sum);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if constexpr (EAGER) {
#pragma unroll
        for (int i = 0; i < 8; ++i) element(cur, 8 * b + i, p, l);
      }
      const v8 pf = pack(p + 8 * b);
      const char* Vb = smem + 2 * TILE + (r + 16 * b) * D * 2;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        acc[d] = El<T>::mma32(join<T>(tr4<T>(reinterpret_cast<const T*>(Vb + vo[d])),
                                      tr4<T>(reinterpret_cast<const T*>(Vb + vu[d]))), pf, acc[d]);
    }
  };
  auto arrive = [&](int j) __attribute__((always_inline)) {   // step j's tiles are there, step j + 1's on their way
    dma_wait<0>();
    if constexpr (Q8) widen(j);             // what the wave itself brought
    __syncthreads();
    if (j < j_end) stage(j + 1);
    if constexpr (!Q8) mend(j);
  };

  if (j_beg < j_end) {
    __syncthreads();                        // the flags are clear
    stage(j_beg);
    int j = j_beg;
    arrive(j);
    if (u_last >= u_beg) {
      f32x16 s0, s1;
      scores(0, s0);
      mask(u_beg, s0);
      follow(maximum(s0));
      if (u_last == u_beg) {
        last_half(s0, 32);
      } else {
        half(u_beg, s0, s1, 0, 1, 32);
        const int jf = (u_last + 1) >> 1;
        ++j;
        if constexpr (!PAGED) {             // two steps, so that the buffers are constants
          for (; j + 1 < jf; j += 2) {      // (over pages the code of two would not fit the cache)
            arrive(j);
            half(2 * j - 1, s1, s0, TILE, 0, 0);
            half(2 * j, s0, s1, TILE, 1, 32);
            arrive(j + 1);
            half(2 * j + 1, s1, s0, 0, 0, 0);
            half(2 * j + 2, s0, s1, 0, 1, 32);
          }
        }
        for (; j < jf; ++j) {
          arrive(j);
          flip();
          half(2 * j - 1, s1, s0, 0, 0, 0);
          half(2 * j, s0, s1, 0, 1, 32);
        }
        arrive(j);
        flip();
        if (u_last & 1) {
          last_half(s1, 0);
        } else {
          half(2 * j - 1, s1, s0, 0, 0, 0);
          last_half(s0, 32);
        }
      }
    }
    for (++j; j <= j_end; ++j) arrive(j);   // other waves' rows see further
  }
  l = pair_sum32(l, l);

  // the lane's row formed again here, not kept in registers through the loop
  int last = threadIdx.x;
  asm volatile("" : "+v"(last));
  const int eh = (last >> 5) & 1, erow = t.row0 + (last >> 6) * 32 + (last & 31);
  const int etok = fdiv(min(erow, t.rows - 1), a.G), ehead = kvh * a.G.d + min(erow, t.rows - 1) - etok * a.G.d;
  const int64_t r = (int64_t)(t.bos + etok) * a.H + ehead;
  char* eo = a.o + (int64_t)(t.bos + etok) * a.o_ts + (int64_t)ehead * a.o_hs + 8 * eh;
  if (PREFIX || a.nsplit > 1) {
    if (erow < t.rows) {
      float* pp = share_row<D>(a, sp, r) + 4 * eh;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(pp + 32 * d + 8 * i) =
              f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
      if (eh == 0) {
        share_stats<D>(a, sp, r)[0] = m * a.c;
        share_stats<D>(a, sp, r)[1] = l;
        if (sp == ns - 1)
          for (int s = ns; s < a.nsplit; ++s) share_stats<D>(a, s, r)[0] = __builtin_bit_cast(float, NO_SHARE);
      }
    }
  } else if (erow < t.rows) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typename El<T>::v4 x;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) x[jj] = (T)(acc[d][4 * i + jj] * inv);
        *reinterpret_cast<typename El<T>::v4*>(eo + 64 * d + 16 * i) = x;
      }
    if (a.lse && eh == 0) a.lse[r] = m * a.c + __builtin_amdgcn_logf(l);
  }
  __syncthreads();
  // the first tile with an edge begins behind wg_first - 63
  if (s_bad && erow < t.rows)
    add_nonfinite<T, D, PAGED, Q8, PREFIX>(a, t, kvh, max(j_beg * BN, off + token_of(t.row0) - 62),
                                           min(j_end * BN, off + (PREFIX ? 0 : etok) + 1), eh, eo,
                                           share_row<D>(a, sp, r) + 4 * eh);
