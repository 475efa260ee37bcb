// Causal softmax attention of whole prompts (contiguous k, v) and of new tokens behind a
// cached context (k, v in pages):
//   s_ij = scale q_i . k_j  (j <= i + keys - tokens),  o_i = sum_j softmax_j(s_ij) v_j
// in one pass over the keys with a running maximum and sum; a row without keys gives 0.
//
// A workgroup of four waves takes 128 rows, 32 to a wave, and walks the keys in tiles of
// 64 staged through LDS (the next tile's loads are in flight while one is computed).
// Rows are (token, head of the group): the heads that share keys sit in one tile, so few
// tokens still fill the 32 columns of a matrix product and the keys are read once for all
// of them.  Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T: a lane
// then holds one row's scores, so the softmax statistics are per-lane scalars and P^T in
// the C layout is already the B operand of the second product (the k order it implies is
// the one the transposing LDS reads of V are made in).
// P is rounded to the inputs' type (half a step of each, averaged over the keys); scores,
// maxima, sums and O stay in fp32.
//
// Bound by the matrix cores and the VALU together: they overlap little (the shares of the
// time that each is at work add up to 100 - 115 %), and the clock falls to 1.6 - 1.8 GHz under
// both, so what pays is fewer instructions.  Measured (a range is that of the cards it was timed
// on): one prompt of 32768, 16 / 4 heads of 128, 3.72 - 4.03 ms, 1.09 - 1.18 PFLOP/s (a large
// matrix product reaches 1.22 - 1.26); packed prompts of 64-wide heads, whose exponentials weigh
// twice as much against their products, 382 - 397 us, 0.83 - 0.86; pieces of prompts over pages
// 842 - 902 us, 0.91 - 0.98; draft tokens of eight sequences to 16384 keys 63 - 75 us and the
// joining 6 (76 us where every sequence's keys were cut into as many splits).
#include "attn.hpp"

namespace hmx {
namespace attn {

constexpr int BM = 128, BN = 64;
constexpr float NO_MC = -1e30f;
constexpr uint32_t NO_SHARE = 0x7fc00000u;   // a NaN, in the place of a share's maximum: there is none

struct FwdArgs {
  const char *q, *k, *v;
  char* o;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;   // bytes
  float* lse;          // [T, H] of the scaled scores in base 2, or NULL
  Seqs seqs;
  Pages pages;
  FastDiv G;
  int32_t H, HKV, slots, fill, nsplit, places;   // nsplit: split.most
  Splits split;
  float c;             // scale log2(e)
  float* part;         // [nsplit][T * H][D], then [nsplit][T * H][2]: maximum and sum
};

// whether a 16-bit value is infinite or NaN, and whether any of eight is
template <typename T> __device__ __forceinline__ bool nonfinite(uint32_t x) {
  constexpr uint32_t E = __is_same(T, bf16) ? 0x7f80u : 0x7c00u;
  return (x & E) == E;
}
template <typename T>
__device__ __forceinline__ bool any_nonfinite(u32x4 x) {
  bool b = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) b |= nonfinite<T>(x[i]) || nonfinite<T>(x[i] >> 16);
  return b;
}
// One key's row of k or v; NULL where its page lies outside the cache.
template <typename T, bool PAGED>
__device__ __forceinline__ const T* key_row(const FwdArgs& a, const Tile& t, int kvh, int j, bool value) {
  if constexpr (PAGED) {
    const int pi = fdiv(j, a.pages.page), pid = a.pages.table[t.seq * a.pages.table_stride + pi];
    if ((unsigned)pid >= (unsigned)a.pages.num_pages) return nullptr;
    const int64_t in = j - pi * a.pages.page.d;
    return reinterpret_cast<const T*>(value ? a.pages.v + pid * a.pages.v_ps + in * a.pages.v_ts + kvh * a.pages.v_hs
                                            : a.pages.k + pid * a.pages.k_ps + in * a.pages.k_ts + kvh * a.pages.k_hs);
  } else {
    return reinterpret_cast<const T*>(value ? a.v + (int64_t)(t.bos + j) * a.v_ts + kvh * a.v_hs
                                            : a.k + (int64_t)(t.bos + j) * a.k_ts + kvh * a.k_hs);
  }
}

// Row `row` of the part over keys k0 .. k1 - 1, unnormalised, in the layout of a split's share.
template <int D>
__device__ __forceinline__ float* share_row(const FwdArgs& a, int sp, int64_t r) {
  return a.part + ((int64_t)sp * a.seqs.T * a.H + r) * D;
}
template <int D>
__device__ __forceinline__ float* share_stats(const FwdArgs& a, int sp, int64_t r) {
  const int64_t n = (int64_t)a.seqs.T * a.H;
  return a.part + (int64_t)a.nsplit * n * D + ((int64_t)sp * n + r) * 2;
}

// What mend() took out of the edge tiles, into the rows that attend it: a value that is not
// finite, times any probability, makes its column of the row that value (two unlike make NaN).
// The lane adds to its part of a row, just stored, from keys k0 .. k1 - 1; where those reach
// tiles that are not at the edge the row has them already, and the same again changes nothing.
// Never reached with finite values.  A prompt of 4096 tokens, 32 / 8 heads of 128, takes 0.42 ms
// with NaN in all values and 0.26 with one row of it, where finite ones take 0.17 (forming the
// tile's rows again key by key took 83 and 40 ms).
template <typename T, int D, bool PAGED>
__device__ __forceinline__ void add_nonfinite(const FwdArgs& a, const Tile& t, int kvh, int k0, int k1, int h,
                                              char* orow, float* share) {
  typedef typename El<T>::v4 v4;
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  constexpr int NV = D / 8;
  f32x4 add[NV];
#pragma unroll
  for (int x = 0; x < NV; ++x) add[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int j = k0; j < k1; ++j) {
    const T* v = key_row<T, PAGED>(a, t, kvh, j, true);
    if (!v) continue;
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const u16x4 b = *reinterpret_cast<const u16x4*>(v + 8 * x + 4 * h);
      const v4 f = __builtin_bit_cast(v4, b);
#pragma unroll
      for (int z = 0; z < 4; ++z) add[x][z] += nonfinite<T>(b[z]) ? (float)f[z] : 0.f;
    }
  }
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    if (add[x][0] == 0.f && add[x][1] == 0.f && add[x][2] == 0.f && add[x][3] == 0.f) continue;
    if (a.nsplit > 1) {
      *reinterpret_cast<f32x4*>(share + 8 * x) += add[x];
    } else {
      v4* o = reinterpret_cast<v4*>(orow + 16 * x);
      v4 y = *o;
#pragma unroll
      for (int z = 0; z < 4; ++z) y[z] = (T)((float)y[z] + add[x][z]);
      *o = y;
    }
  }
}

// The loop is software-pipelined by halves of 32 keys: while a half's probabilities are
// formed in the VALU, the matrix cores form the next half's scores, then its product with V
// while the second sixteen probabilities and the next half's maximum are formed.  A step of
// the loop multiplies K's keys 64 j .. 64 j + 63 and V's 64 j - 32 .. 64 j + 31, so both
// tiles have two buffers, and arrive in LDS directly, a step ahead of their use.
// Workgroups of a compute unit: two at head size 128, for the registers; at 64 three, which
// hides more of the exponentials (404 -> 396 us on packed prompts).  Outside the loop registers
// spill: 50 at 128 and 38 at 64 over contiguous keys, 4 and 6 over pages.
template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_fwd_kernel(FwdArgs a) {
  typedef typename El<T>::v8 v8;
  constexpr int NC = D / 8;                 // 16-byte chunks of a row
  constexpr int RI = 64 / NC, NL = 16 / RI; // rows of a wave's load, loads of its 16 rows of a tile
  constexpr int NS = D / 16, ND = D / 32;
  constexpr int TILE = BN * D * 2;          // bytes
  __shared__ __align__(1024) char smem[4 * TILE];   // K, K, V, V
  __shared__ int s_bad, s_skip[4];

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // uniform, and known to be
  const int kvh = blockIdx.x % a.HKV;
  const Tile t = next_tile<BM, true>(a.seqs, PAGED ? a.pages.lens : nullptr, place(blockIdx.x / a.HKV, gridDim.x / a.HKV, a.places), a.slots,
                                       a.split);
  if (t.row0 >= t.rows || t.row0 < 0) return;

  const int row = t.row0 + wave * 32 + l32;
  const int rowc = min(row, t.rows - 1);
  const int tok = fdiv(rowc, a.G), head = kvh * a.G.d + rowc - tok * a.G.d;
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
  const int off = keys - t.tokens;          // token i attends keys 0 .. off + i
  const int klast = off + tok;
  const int wrow = t.row0 + wave * 32;
  const int w_first = off + fdiv(min(wrow, t.rows - 1), a.G);            // least last key of the wave's rows
  const int w_last = off + fdiv(min(wrow + 31, t.rows - 1), a.G);        // and greatest
  const int wg_first = off + fdiv(t.row0, a.G);
  const int wg_last = off + fdiv(min(t.row0 + BM, t.rows) - 1, a.G);
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
  auto stage = [&](int j) __attribute__((always_inline)) {                 // the keys and values of step j
    if (j < j_end) stage_rows(j, j * BN + wave * 16, false);
    stage_rows(j, j * BN - 32 + wave * 16, true);
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
    __syncthreads();
    if (j < j_end) stage(j + 1);
    mend(j);
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
  if (a.nsplit > 1) {
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
    add_nonfinite<T, D, PAGED>(a, t, kvh, max(j_beg * BN, off + fdiv(t.row0, a.G) - 62), min(j_end * BN, off + etok + 1),
                               eh, eo, share_row<D>(a, sp, r) + 4 * eh);
}

// The splits' shares of a row joined: sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.  The
// tokens of all sequences lie between the first and the last offset.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(FwdArgs a) {
  constexpr int TPR = D / 4;
  const int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int tok = (int)(r / a.H), h = (int)(r - (int64_t)tok * a.H), d = 4 * (threadIdx.x % TPR);
  if (tok >= a.seqs.T || (a.seqs.cu && (tok < a.seqs.cu[0] || tok >= a.seqs.cu[a.seqs.N]))) return;
  int ns = 0;
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) ns += __builtin_bit_cast(uint32_t, share_stats<D>(a, s, r)[0]) != NO_SHARE;
  float m = NEG_INF, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < ns; ++s) {
    const float* st = share_stats<D>(a, s, r);
    const f32x4 x = *reinterpret_cast<const f32x4*>(share_row<D>(a, s, r) + d);
    const float mn = fmaxf(m, st[0]), ref = mn == NEG_INF ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(st[0] - ref);
    l = l * f + e * st[1];
    o = o * f + x * e;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  typename El<T>::v4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (T)(o[i] * inv);
  *reinterpret_cast<typename El<T>::v4*>(a.o + (int64_t)tok * a.o_ts + (int64_t)h * a.o_hs + 2 * d) = x;
  if (a.lse && d == 0) a.lse[r] = m + __builtin_amdgcn_logf(l);
}

// Splits of the keys, where the row tiles alone leave compute units idle: as many as give each
// about two workgroups (what runs at once).  A split costs its share's trip through memory and
// the joining launch, so it has at least `least` tiles of keys: four over pages, where there
// are few rows, eight over contiguous keys.  A tile of a longer sequence may take twice as many.
// Prompts, without splits and with: 2048 tokens, 8 / 2 heads of 128, 42.5 -> 31.6 us; 4096,
// 4 / 4 of 64, 58 -> 28; 16384, 2 / 1 of 128, 276 -> 175.
static Splits splits(int64_t tiles, int HKV, int64_t max_keys, int least) {
  const int64_t live = tiles * HKV, want = 2ll * cu_count(), most = max_keys / (least * BN);
  int64_t even = live > 0 ? want / live : 1;
  if (even > most) even = most;
  if (even > 64) even = 64;
  if (even <= 1) return NO_SPLITS;
  return Splits{(int32_t)even, (int32_t)(2 * even < most ? 2 * even : most), (int32_t)(want / HKV), least};
}

template <typename T, bool PAGED>
static void launch_fwd(FwdArgs a, int D, hipStream_t s) {
  a.places = (int32_t)(cu_count() / a.HKV);
  int64_t blocks = a.slots;                 // of a kv head
  if (a.nsplit > 1) blocks = !a.seqs.cu || a.seqs.N > LANE_SEQS ? blocks * a.split.even : blocks + a.split.blocks;
  const dim3 grid((unsigned)(blocks * a.HKV));
  if (D == 64) hipLaunchKernelGGL((attn_fwd_kernel<T, 64, PAGED>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((attn_fwd_kernel<T, 128, PAGED>), grid, dim3(256), 0, s, a);
  if (a.nsplit > 1) {
    const int64_t rows = (int64_t)a.seqs.T * a.H, rpb = 1024 / D;
    const dim3 jg((unsigned)((rows + rpb - 1) / rpb));
    if (D == 64) hipLaunchKernelGGL((attn_join_kernel<T, 64>), jg, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_join_kernel<T, 128>), jg, dim3(256), 0, s, a);
  }
}

}  // namespace attn
}  // namespace hmx

using namespace hmx;

#define ATTN_COMMON_CHECKS(what)                                                                    HMX_REQUIRE(D == 64 || D == 128, HMX_EUNSUPPORTED, what ": head size %d not in {64, 128}", D);    HMX_REQUIRE(dtype == HMX_BF16 || dtype == HMX_F16, HMX_EUNSUPPORTED,                                          what ": dtype code %d (bf16 or fp16)", dtype);                                        HMX_REQUIRE(N >= 0 && T >= 0 && HKV > 0 && H > 0 && H % HKV == 0, HMX_EINVAL,                                 what ": N=%d T=%lld H=%d HKV=%d", N, (long long)T, H, HKV);                           HMX_REQUIRE(T * (H / HKV) < (1ll << 30), HMX_EUNSUPPORTED, what ": %lld tokens", (long long)T);   HMX_REQUIRE(scale > 0.f && scale < __builtin_inff(), HMX_EINVAL, what ": scale %g must be positive", (double)scale);

// Packed lengths are on the device: the longest sequence is taken to be at most four times
// their mean (many short prompts are not split, nor sent through a workspace for it), and
// more sequences than next_tile can weigh are not split.
static attn::Splits prompt_splits(int64_t N, int64_t T, int H, int HKV, bool packed) {
  if (N <= 0 || T <= 0 || (packed && N > attn::LANE_SEQS)) return attn::NO_SPLITS;
  const int32_t some = 0;
  const int64_t slots = attn::tile_slots<attn::BM>(packed ? &some : nullptr, N, T, H / HKV);
  return attn::splits(packed ? slots - 2 : slots, HKV, packed && N <= 4 ? T : packed ? 4 * T / N : T / N, 8);
}

extern "C" size_t hmx_causal_attention_workspace_bytes(int32_t N, int64_t T, int32_t H, int32_t HKV,
                                                       int32_t D, int32_t packed) {
  if (N <= 0 || T <= 0 || HKV <= 0 || H <= 0 || H % HKV != 0) return 0;
  const int ns = prompt_splits(N, T, H, HKV, packed != 0).most;
  return ns == 1 ? 0 : (size_t)ns * T * H * (D + 2) * sizeof(float);
}

extern "C" int hmx_causal_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                    const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                    const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                    int32_t dtype, void* o, int64_t o_token_stride,
                                    int64_t o_head_stride, float* lse, const int32_t* cu_seqlens,
                                    int32_t N, int64_t T, int32_t H, int32_t HKV, int32_t D,
                                    float scale, int32_t fill_gaps, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  ATTN_COMMON_CHECKS("hmx_causal_attention")
  HMX_REQUIRE(cu_seqlens || N == 0 || T % N == 0, HMX_EINVAL, "hmx_causal_attention: T=%lld is not N=%d sequences",
              (long long)T, N);
  if (T == 0 || (N == 0 && !cu_seqlens)) return HMX_OK;
  HMX_REQUIRE(q && k && v && o, HMX_EINVAL, "hmx_causal_attention: null pointer");
  const int64_t st = q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride |
                     v_head_stride | o_token_stride | o_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0, HMX_EINVAL,
              "hmx_causal_attention: strides must be multiples of 8 elements and pointers 16-byte aligned");
  HMX_REQUIRE(attn::near_rows(k_token_stride) && attn::near_rows(v_token_stride), HMX_EUNSUPPORTED,
              "hmx_causal_attention: token strides of k and v past 2^25 elements");
  attn::FwdArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.o = (char*)o;
  a.q_ts = 2 * q_token_stride; a.q_hs = 2 * q_head_stride;
  a.k_ts = 2 * k_token_stride; a.k_hs = 2 * k_head_stride;
  a.v_ts = 2 * v_token_stride; a.v_hs = 2 * v_head_stride;
  a.o_ts = 2 * o_token_stride; a.o_hs = 2 * o_head_stride;
  a.lse = lse;
  a.seqs = attn::Seqs{cu_seqlens, N, (int32_t)T, H / HKV};
  a.G = attn::fast_div(H / HKV);
  const int64_t slots = attn::tile_slots<attn::BM>(cu_seqlens, N, T, H / HKV);
  HMX_REQUIRE(slots * HKV < (1ll << 31), HMX_EUNSUPPORTED, "hmx_causal_attention: %lld tiles", (long long)slots);
  a.H = H; a.HKV = HKV; a.slots = (int32_t)slots; a.fill = fill_gaps;
  a.split = prompt_splits(N, T, H, HKV, cu_seqlens != nullptr);
  a.nsplit = a.split.most;
  a.part = static_cast<float*>(workspace);
  HMX_REQUIRE(a.nsplit == 1 ||
                  (workspace && (uintptr_t)workspace % 16 == 0 &&
                   workspace_bytes >= hmx_causal_attention_workspace_bytes(N, T, H, HKV, D, cu_seqlens != nullptr)),
              HMX_EINVAL, "hmx_causal_attention: workspace of %zu bytes is too small", workspace_bytes);
  a.c = scale * attn::LOG2E;
  if (dtype == HMX_BF16) attn::launch_fwd<bf16, false>(a, D, (hipStream_t)stream);
  else attn::launch_fwd<f16, false>(a, D, (hipStream_t)stream);
  return check_launch("hmx_causal_attention");
}

static attn::Splits paged_splits(int64_t N, int64_t T, int H, int HKV, int64_t max_keys) {
  const int32_t packed = 0;
  return attn::splits(attn::tile_slots<attn::BM>(&packed, N, T, H / HKV) - 2, HKV, max_keys, 4);
}

extern "C" size_t hmx_paged_causal_attention_workspace_bytes(int32_t N, int64_t T, int32_t H,
                                                             int32_t HKV, int32_t D,
                                                             int64_t max_keys) {
  if (N <= 0 || T <= 0 || HKV <= 0 || H <= 0 || H % HKV != 0) return 0;
  const int ns = paged_splits(N, T, H, HKV, max_keys).most;
  return ns == 1 ? 0 : (size_t)ns * T * H * (D + 2) * sizeof(float);
}

extern "C" int hmx_paged_causal_attention(const void* q, int64_t q_token_stride,
                                          int64_t q_head_stride, int32_t dtype, void* o,
                                          int64_t o_token_stride, int64_t o_head_stride,
                                          const hmx_paged_kv* cache, const int32_t* cu_seqlens,
                                          int32_t N, int64_t T, int32_t H, int32_t HKV, int32_t D,
                                          float scale, int32_t fill_gaps, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  ATTN_COMMON_CHECKS("hmx_paged_causal_attention")
  HMX_REQUIRE(cache && cache->num_pages >= 0 && cache->page_size > 0 && cache->table_width >= 0, HMX_EINVAL,
              "hmx_paged_causal_attention: cache");
  if (T == 0) return HMX_OK;
  HMX_REQUIRE(q && o && cu_seqlens && (N == 0 || (cache->seq_lens && attn::has_pages(*cache))),
              HMX_EINVAL, "hmx_paged_causal_attention: null pointer");
  const int64_t max_keys = (int64_t)cache->table_width * cache->page_size;
  HMX_REQUIRE(max_keys < (1ll << 31) - 256, HMX_EUNSUPPORTED,
              "hmx_paged_causal_attention: a table row holds %lld keys", (long long)max_keys);
  const int64_t st = q_token_stride | q_head_stride | o_token_stride | o_head_stride |
                     cache->k_page_stride | cache->k_token_stride | cache->k_head_stride |
                     cache->v_page_stride | cache->v_token_stride | cache->v_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)o | (uintptr_t)cache->k | (uintptr_t)cache->v;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0, HMX_EINVAL,
              "hmx_paged_causal_attention: strides must be multiples of 8 elements and pointers 16-byte aligned");
  HMX_REQUIRE(attn::near_rows(cache->k_token_stride) && attn::near_rows(cache->v_token_stride), HMX_EUNSUPPORTED,
              "hmx_paged_causal_attention: token strides of the cache past 2^25 elements");
  attn::FwdArgs a{};
  a.q = (const char*)q; a.o = (char*)o;
  a.q_ts = 2 * q_token_stride; a.q_hs = 2 * q_head_stride;
  a.o_ts = 2 * o_token_stride; a.o_hs = 2 * o_head_stride;
  a.seqs = attn::Seqs{cu_seqlens, N, (int32_t)T, H / HKV};
  a.G = attn::fast_div(H / HKV);
  a.pages = attn::make_pages(*cache);
  const int64_t slots = attn::tile_slots<attn::BM>(cu_seqlens, N, T, H / HKV);
  HMX_REQUIRE(slots * HKV < (1ll << 31), HMX_EUNSUPPORTED, "hmx_paged_causal_attention: %lld tiles",
              (long long)slots);
  a.H = H; a.HKV = HKV; a.slots = (int32_t)slots; a.fill = fill_gaps;
  a.split = N == 0 ? attn::NO_SPLITS : paged_splits(N, T, H, HKV, max_keys);
  a.nsplit = a.split.most;
  a.part = static_cast<float*>(workspace);
  HMX_REQUIRE(a.nsplit == 1 ||
                  (workspace && (uintptr_t)workspace % 16 == 0 &&
                   workspace_bytes >= hmx_paged_causal_attention_workspace_bytes(N, T, H, HKV, D, max_keys)),
              HMX_EINVAL, "hmx_paged_causal_attention: workspace of %zu bytes is too small", workspace_bytes);
  a.c = scale * attn::LOG2E;
  if (dtype == HMX_BF16) attn::launch_fwd<bf16, true>(a, D, (hipStream_t)stream);
  else attn::launch_fwd<f16, true>(a, D, (hipStream_t)stream);
  return check_launch("hmx_paged_causal_attention");
}
