// The backward of causal attention.  With P = exp2(c q.k - lse) (lse from the forward),
// dP = dO V^T, delta_i = dO_i . O_i and dS = P (dP - delta):
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO   (summed over a group's heads)
//
// Two kernels, so that every gradient is summed in one workgroup's registers in one order:
// dQ by row tiles (which also forms delta), dK and dV by key tiles over the rows of all
// heads of the group.  S and dP are formed in both: seven products instead of five, in
// exchange for no atomics, no fp32 copy of dQ in memory and the same result every time.
// Products are transposed where that leaves P and dS as B operands in the C layout.
// P and dS are rounded to bf16 (half a step, as the inputs themselves are); everything
// else stays in fp32.  What that costs against float64, where rounding the results alone makes
// an error of 1.7e-3: dV 2.3e-3, dK 2.4e-3, dQ 2.4 - 2.5e-3.  delta is formed from the rounded
// O, and in rows that attend few keys its error, times P K, was more than all others together
// (dQ 2.8 - 3.0e-3, up to 3.9e-3 in short sequences).  Since dS sums to 0, what it does sum to
// is that error: dK's delta is put right by it, and dQ by it times the greatest P's keys.
// Looking for those costs nothing measurable where no P passes 1/8, 1 - 2 % of the step in
// peaked heads, 8 % at 512 tokens.  Eight more bits of O beside it took dQ's error to 2.6e-3
// for 1.2 % of the step and half as much memory again as O's; dS in two parts would take its
// rounding away too, for one more product.  Neither is done.
//
// Measured at 8 x 4096 tokens, 32 / 8 heads of 128 (forward 1.06 ms): dQ 1.55 ms, 1.07 PFLOP/s;
// dK and dV 2.33 ms, 0.94; a large matrix product reaches 1.22 - 1.26.
#include "attn.hpp"

#include <type_traits>

namespace hmx {
namespace attn {

struct BwdArgs {
  const char *q, *k, *v, *o, *dout;
  char *dq, *dk, *dv;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs, do_ts, do_hs;   // bytes
  int64_t dq_ts, dq_hs, dk_ts, dk_hs, dv_ts, dv_hs;
  const float* lse;    // [T, H]
  float* delta;        // [T, H]
  Seqs seqs;           // rows of tokens x G
  FastDiv G;
  int32_t H, HKV, slots;
  int32_t fixed;       // a tile's rows lie at fixed 32-bit offsets (unsigned) from its first token
  float c, scale;
};

constexpr int QM = 128;              // dQ: rows of a workgroup

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void attn_bwd_dq_kernel(BwdArgs a) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int QN = 64;                    // keys of a tile
  constexpr int NC = D / 8, RI = 64 / NC, NL = 16 / RI, NS = D / 16, ND = D / 32;
  __shared__ __align__(16) T Ks[2][QN * D];
  __shared__ __align__(16) T Vs[2][QN * D];

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // uniform, and known to be
  const int kvh = blockIdx.x % a.HKV;
  const Tile t = next_tile<QM, true>(a.seqs, nullptr, blockIdx.x / a.HKV, a.slots);
  if (t.row0 >= t.rows || t.row0 < 0) return;
  const int row = t.row0 + wave * 32 + l32, rowc = min(row, t.rows - 1);
  const int tok = fdiv(rowc, a.G), head = kvh * a.G.d + rowc - tok * a.G.d;
  const int64_t gt = t.bos + tok;
  char* dqr = a.dq + gt * a.dq_ts + (int64_t)head * a.dq_hs;
  if (t.seq < 0) {                          // rows of no sequence
    if (row < t.rows)
#pragma unroll
      for (int i = 0; i < NS; ++i) *reinterpret_cast<u32x4*>(dqr + 32 * i + 16 * h) = u32x4{0, 0, 0, 0};
    return;
  }
  const int wrow = t.row0 + wave * 32;
  const int w_first = fdiv(min(wrow, t.rows - 1), a.G), w_last = fdiv(min(wrow + 31, t.rows - 1), a.G);
  const int nt = fdiv(min(t.row0 + QM, t.rows) - 1, a.G) / QN + 1;
  const int keys = t.tokens;

  v8 qf[NS], df[NS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = *reinterpret_cast<const v8*>(a.q + gt * a.q_ts + (int64_t)head * a.q_hs + 32 * s + 16 * h);
    df[s] = *reinterpret_cast<const v8*>(a.dout + gt * a.do_ts + (int64_t)head * a.do_hs + 32 * s + 16 * h);
    const v8 of = *reinterpret_cast<const v8*>(a.o + gt * a.o_ts + (int64_t)head * a.o_hs + 32 * s + 16 * h);
#pragma unroll
    for (int i = 0; i < 8; ++i) delta += (float)df[s][i] * (float)of[i];
  }
  delta = pair_sum32(delta, delta);
  const float lse = a.lse[gt * a.H + head];
  float over = 0.f;                         // the sum of dS, own half's keys
  // the own half's greatest P past 1/8, its place among the 16 of a unit in the low bits, and the unit
  uint32_t top = __builtin_bit_cast(uint32_t, 0.125f) | 15;
  int top_unit = -1;

  // staging as in the forward: the wave brings rows 16 wave .. 16 wave + 15 of a tile
  uint32_t koff[NL], voff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = i * RI + lane / NC, c = swz<D>(wave * 16 + r, lane % NC);
    koff[i] = (uint32_t)(r * (int)a.k_ts + 16 * c);
    voff[i] = (uint32_t)(r * (int)a.v_ts + 16 * c);
  }
  const char* kbase = a.k + (int64_t)t.bos * a.k_ts + (int64_t)kvh * a.k_hs;
  const char* vbase = a.v + (int64_t)t.bos * a.v_ts + (int64_t)kvh * a.v_hs;
  auto stage = [&](int j) __attribute__((always_inline)) {
    const uint32_t kl = lds_addr(Ks[j & 1]) + wave * 16 * D * 2, vl = lds_addr(Vs[j & 1]) + wave * 16 * D * 2;
    const int r0 = j * QN + wave * 16;
    if (r0 + 16 <= keys) {
      const char *kb = uniform_ptr(kbase + r0 * a.k_ts), *vb = uniform_ptr(vbase + r0 * a.v_ts);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(kl + i * RI * D * 2, kb, koff[i]);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(vl + i * RI * D * 2, vb, voff[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int x = i * RI + lane / NC, r = min(r0 + x, keys - 1), c = 16 * swz<D>(wave * 16 + x, lane % NC);
        dma16(kl + i * RI * D * 2, kbase + r * a.k_ts + c);
        dma16(vl + i * RI * D * 2, vbase + r * a.v_ts + c);
      }
    }
  };
  int ko[NS], to[ND], tu[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s) ko[s] = l32 * D + swz<D>(l32, 2 * s + h) * 8;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    to[d] = tr_offset<D>(lane, d, false);
    tu[d] = tr_offset<D>(lane, d, true);
  }
  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x16{0};

  auto step = [&](int j, int buf) __attribute__((always_inline)) {
    const T *Kb = Ks[buf], *Vb = Vs[buf];
    dma_wait<0>();
    __syncthreads();
    if (j + 1 < nt) stage(j + 1);
    const int t0 = j * QN;
    if (t0 > w_last) return;
#pragma unroll
    for (int kt = 0; kt < QN / 32; ++kt) {
      f32x16 st = {0}, dp = {0};
#pragma unroll
      for (int s = 0; s < NS; ++s)
        st = El<T>::mma32(*reinterpret_cast<const v8*>(Kb + ko[s] + kt * 32 * D), qf[s], st);
#pragma unroll
      for (int s = 0; s < NS; ++s)
        dp = El<T>::mma32(*reinterpret_cast<const v8*>(Vb + ko[s] + kt * 32 * D), df[s], dp);
      if (t0 + kt * 32 + 31 > w_first) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t0 + kt * 32 + 8 * (i >> 2) + 4 * h + (i & 3) > tok) st[i] = NEG_INF;
      }
      uint32_t p[16];                       // P, as the bits of positive numbers
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_exp2f(st[i] * a.c - lse));
      uint32_t mx = max(p[0], p[1]);
#pragma unroll
      for (int i = 2; i < 16; ++i) mx = max(mx, p[i]);
      if (__any(mx > top)) {
        mx = p[0] & ~15u;
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = max(mx, (p[i] & ~15u) | (uint32_t)i);
        if (mx > top) {
          top = mx;
          top_unit = 2 * j + kt;
        }
      }
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        ds[i] = __builtin_bit_cast(float, p[i]) * (dp[i] - delta);
        over += ds[i];
      }
      const v8 d0 = pack8<T>(ds[0], ds[1], ds[2], ds[3], ds[4], ds[5], ds[6], ds[7]);
      const v8 d1 = pack8<T>(ds[8], ds[9], ds[10], ds[11], ds[12], ds[13], ds[14], ds[15]);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const T* kp = Kb + (kt * 32 + ks * 16) * D;
          acc[d] = El<T>::mma32(join<T>(tr4<T>(kp + to[d]), tr4<T>(kp + tu[d])), ks ? d1 : d0, acc[d]);
        }
    }
  };
  stage(0);
  for (int j = 0; j < nt; j += 2) {         // two steps, so that the buffers are constants
    step(j, 0);
    if (j + 1 < nt) step(j + 1, 1);
  }
  // P sums to 1, so dS would sum to 0 had delta been formed from an exact O: what it does
  // sum to is delta's error, and dK gets a delta without it.
  over = pair_sum32(over, over);
  if (h == 0 && row < t.rows) a.delta[gt * a.H + head] = delta + over;
  // dQ has -delta's error times P K.  P K would be another product, but where it is not small
  // most of it is the greatest probabilities' keys, one of either half's: those are taken out.
  const float w = top_unit < 0 ? 0.f : over * __builtin_bit_cast(float, top & ~15u);
  // (clamped: where the row's own scores are NaN so is P behind its last key)
  const int top_key = min(max(top_unit, 0) * 32 + 8 * (int)((top & 15) >> 2) + 4 * h + (int)(top & 3), tok);
  const float w_other = shfl_xor(w, 32);
  const int key_other = __shfl_xor(top_key, 32, 64);
#pragma unroll 1
  for (int x = 0; x < 2; ++x) {
    const float wx = x ? w_other : w;
    if (wx == 0.f) continue;
    const T* kp = reinterpret_cast<const T*>(kbase + (x ? key_other : top_key) * a.k_ts) + 4 * h;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v4 kv = *reinterpret_cast<const v4*>(kp + 32 * d + 8 * i);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) acc[d][4 * i + jj] -= wx * (float)kv[jj];
      }
  }
  if (row < t.rows) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4 x;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) x[jj] = (T)(acc[d][4 * i + jj] * a.scale);
        *reinterpret_cast<v4*>(dqr + (32 * d + 8 * i + 4 * h) * 2) = x;
      }
  }
}

constexpr int KM = 128, KR = 64;     // dK, dV: keys of a workgroup, rows of a tile

// A wave holds 32 keys: their K and V rows as B operands and dK^T, dV^T as accumulators in
// registers (one wave a SIMD), and walks the rows that see them.  Pipelined by units
// of 32 rows: S and dP of the next unit are formed by the matrix cores while P and dS of
// this one are formed in the VALU.  Tiles of 64 rows of Q and dO arrive in LDS directly, in
// a ring of four, two tiles ahead: a step still multiplies with the last unit of the tile
// before (with one tile ahead 5 % slower).  The sums, 128 registers of a wave, and its K and V, 64,
// are why there is one wave a SIMD; sharing P between two waves through LDS instead, so that
// each keeps half of it, took 2.60 ms where this takes 2.47.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void attn_bwd_dkv_kernel(BwdArgs a) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int NC = D / 8, RI = 64 / NC, NL = 16 / RI, NS = D / 16, ND = D / 32;
  constexpr int TILE = KR * D * 2;          // bytes
  constexpr int RING = 4;
  __shared__ __align__(1024) char smem[RING * 2 * TILE];  // [RING][Q, dO]
  __shared__ __align__(16) float Ls[RING][2][KR];         // lse and delta of the rows

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.HKV;
  Seqs sk = a.seqs;
  sk.G = 1;
  const Tile t = next_tile<KM, false>(sk, nullptr, blockIdx.x / a.HKV, a.slots);
  if (t.row0 >= t.rows || t.row0 < 0) return;
  const int key = t.row0 + wave * 32 + l32, keyc = min(key, t.tokens - 1);
  const int64_t gk = t.bos + keyc;
  char* dkr = a.dk + gk * a.dk_ts + (int64_t)kvh * a.dk_hs;
  char* dvr = a.dv + gk * a.dv_ts + (int64_t)kvh * a.dv_hs;
  if (t.seq < 0) {
    if (key < t.tokens)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        *reinterpret_cast<u32x4*>(dkr + 32 * i + 16 * h) = u32x4{0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(dvr + 32 * i + 16 * h) = u32x4{0, 0, 0, 0};
      }
    return;
  }
  v8 kf[NS], vf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    kf[s] = *reinterpret_cast<const v8*>(a.k + gk * a.k_ts + (int64_t)kvh * a.k_hs + 32 * s + 16 * h);
    vf[s] = *reinterpret_cast<const v8*>(a.v + gk * a.v_ts + (int64_t)kvh * a.v_hs + 32 * s + 16 * h);
  }
  const int G = a.G.d, rows = t.tokens * G, nt = (rows + KR - 1) / KR;
  const int wk0 = min(t.row0 + wave * 32, t.tokens - 1);           // the wave's first key
  const int j_wg = t.row0 * G / KR, j_own = wk0 * G / KR;          // first tiles with rows that see them
  const int first = key * G;                                        // the key's first row

  // Staging: rows 16 wave .. + 15 of a tile, RI to a load.  Where G divides a tile's rows, a
  // lane's rows of all tiles are one head's, at offsets that do not change.
  uint32_t qoff[NL], ooff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int x = wave * 16 + i * RI + lane / NC, tk = fdiv(x, a.G), g = x - tk * G;
    const int c = swz<D>(x, lane % NC);
    qoff[i] = (uint32_t)(tk * a.q_ts + g * a.q_hs + 16 * c);
    ooff[i] = (uint32_t)(tk * a.do_ts + g * a.do_hs + 16 * c);
  }
  const char* qbase = a.q + (int64_t)t.bos * a.q_ts + (int64_t)kvh * G * a.q_hs;
  const char* obase = a.dout + (int64_t)t.bos * a.do_ts + (int64_t)kvh * G * a.do_hs;
  const int tpt = KR / G;                   // tokens of a tile where G divides it
  auto stage = [&](int j, int buf) __attribute__((always_inline)) {
    const uint32_t ql = lds_addr(smem) + buf * 2 * TILE + wave * 16 * D * 2, ol = ql + TILE;
    if (a.fixed && (j + 1) * KR <= rows) {
      const char *qb = uniform_ptr(qbase + (int64_t)j * tpt * a.q_ts), *ob = uniform_ptr(obase + (int64_t)j * tpt * a.do_ts);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(ql + i * RI * D * 2, qb, qoff[i]);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(ol + i * RI * D * 2, ob, ooff[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int x = wave * 16 + i * RI + lane / NC, r = min(j * KR + x, rows - 1), tk = fdiv(r, a.G);
        const int g = r - tk * G, c = 16 * swz<D>(x, lane % NC);
        dma16(ql + i * RI * D * 2, qbase + tk * a.q_ts + g * a.q_hs + c);
        dma16(ol + i * RI * D * 2, obase + tk * a.do_ts + g * a.do_hs + c);
      }
    }
    const int r = min(j * KR + lane, rows - 1), tk = fdiv(r, a.G);   // wave 0 (and 2) lse, 1 (and 3) delta
    dma4(lds_addr(&Ls[buf][wave & 1][0]), reinterpret_cast<const char*>(
        ((wave & 1) ? a.delta : a.lse) + ((int64_t)(t.bos + tk) * a.H + kvh * G + r - tk * G)));
  };
  int qo[NS], to[ND], tu[ND];               // byte offsets into a tile
#pragma unroll
  for (int s = 0; s < NS; ++s) qo[s] = (l32 * D + swz<D>(l32, 2 * s + h) * 8) * 2;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    to[d] = tr_offset<D>(lane, d, false) * 2;
    tu[d] = tr_offset<D>(lane, d, true) * 2;
  }
  f32x16 ak[ND], av[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) ak[i] = av[i] = f32x16{0};

  auto mask = [&](int u, f32x16& st) __attribute__((always_inline)) {
    // rows before the key do not see it, and rows behind the last are none
    if (u * 32 < (wk0 + 31) * G || u * 32 + 32 > rows) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = u * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (r < first || r >= rows) st[i] = NEG_INF;
      }
    }
  };
  // The two parts of a unit's work that the pipeline keeps apart: S and dP of unit xn of the
  // tile in bn (NEXT), and P, dS and their products for unit xc of the tile in bc, whose S
  // and dP are st and dp (THIS); together, the first part's products hide the second's
  // exponentials.  LDS reads run AHEAD steps before their use, also into the unit that is
  // NEXT in the following call (FOLLOW: unit xf of the tile in bf).
  constexpr int AHEAD = NS / 2;
  constexpr int E = 16 / NS;                // elements of P formed beside a step of the first part
  v8 qa[NS], oa[NS];
  f32x4 le[4], dl[4];
  auto rows_of = [&](int buf, int x, int s) __attribute__((always_inline)) {
    const char* q = smem + buf * 2 * TILE + x * 32 * D * 2;
    qa[s] = *reinterpret_cast<const v8*>(q + qo[s]);
    oa[s] = *reinterpret_cast<const v8*>(q + TILE + qo[s]);
  };
  auto work = [&](auto NEXT, auto THIS, auto FOLLOW, int bn, int xn, f32x16& sn, f32x16& dn, int bc, int xc,
                  const f32x16& st, const f32x16& dp, int bf, int xf) __attribute__((always_inline)) {
    constexpr bool next = decltype(NEXT)::value, cur = decltype(THIS)::value, follow = decltype(FOLLOW)::value;
    const char *qc = smem + bc * 2 * TILE + xc * 32 * D * 2, *oc = qc + TILE;
    v8 qt[2 * ND], ot[2 * ND], pf[2], sf[2];
    float p[16], ds[16];
    auto cols_of = [&](int g) __attribute__((always_inline)) {
      const int d = g % ND, at = (g / ND) * 16 * D * 2;
      ot[g] = join<T>(tr4<T>(reinterpret_cast<const T*>(oc + to[d] + at)), tr4<T>(reinterpret_cast<const T*>(oc + tu[d] + at)));
      qt[g] = join<T>(tr4<T>(reinterpret_cast<const T*>(qc + to[d] + at)), tr4<T>(reinterpret_cast<const T*>(qc + tu[d] + at)));
    };
    auto pack = [&](int b) __attribute__((always_inline)) {
      const int z = 8 * b;
      pf[b] = pack8<T>(p[z], p[z + 1], p[z + 2], p[z + 3], p[z + 4], p[z + 5], p[z + 6], p[z + 7]);
      sf[b] = pack8<T>(ds[z], ds[z + 1], ds[z + 2], ds[z + 3], ds[z + 4], ds[z + 5], ds[z + 6], ds[z + 7]);
    };
    fence();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (next) {
        if (s + AHEAD < NS) rows_of(bn, xn, s + AHEAD);
      }
      if constexpr (cur) {
        if (s + AHEAD >= NS) cols_of(s + AHEAD - NS);
      }
      if constexpr (next) {
        sn = El<T>::mma32(qa[s], kf[s], s == 0 ? f32x16{0} : sn);
        dn = El<T>::mma32(oa[s], vf[s], s == 0 ? f32x16{0} : dn);
      }
      if constexpr (cur) {
#pragma unroll
        for (int e = s * E; e < s * E + E; ++e) {
          p[e] = __builtin_amdgcn_exp2f(st[e] * a.c - le[e >> 2][e & 3]);
          ds[e] = p[e] * (dp[e] - dl[e >> 2][e & 3]);
        }
        if (s == NS / 2 - 1) pack(0);
        if (s == NS - 1) pack(1);
      }
      fence();
    }
#pragma unroll
    for (int g = 0; g < 2 * ND; ++g) {
      if constexpr (cur) {
        if (g + AHEAD < 2 * ND) cols_of(g + AHEAD);
      }
      if constexpr (follow) {
        if (g >= 2 * ND - AHEAD) rows_of(bf, xf, g - 2 * ND + AHEAD);
      }
      if constexpr (next) {                 // the row terms of the unit that is THIS in the following call
        if (g < 4) {
          const float* ls = &Ls[bn][0][xn * 32 + 4 * h];
          le[g] = *reinterpret_cast<const f32x4*>(ls + 8 * g);
          dl[g] = *reinterpret_cast<const f32x4*>(ls + KR + 8 * g);
        }
      }
      if constexpr (cur) {
        av[g % ND] = El<T>::mma32(ot[g], pf[g / ND], av[g % ND]);
        ak[g % ND] = El<T>::mma32(qt[g], sf[g / ND], ak[g % ND]);
      }
      fence();
    }
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};

  f32x16 s0, d0, s1, d1;
  int buf = RING - 1, next = 0;             // of the tile at work, and of the one after it
  auto arrive = [&](int j) __attribute__((always_inline)) {   // tile j is there, the RING - 2 after it on their way
    if (j + RING - 3 < nt) dma_wait<(RING - 3) * (2 * NL + 1)>();
    else dma_wait<0>();
    __syncthreads();
    if (j + RING - 2 < nt) stage(j + RING - 2, (next + RING - 2) % RING);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    buf = next;
    next = (next + 1) % RING;
  };
  int j = j_wg;
#pragma unroll
  for (int i = 0; i < RING - 2; ++i)
    if (j + i < nt) stage(j + i, i);
  for (; j <= j_own; ++j) {                 // rows before the wave's keys
    arrive(j);
    advance();
  }
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) rows_of(buf, 0, s);
  work(yes, no, yes, buf, 0, s0, d0, buf, 0, s0, d0, buf, 1);
  for (; j < nt; ++j) {                     // tile j - 1, with the beginning of tile j
    mask(2 * j - 2, s0);
    arrive(j);
    work(yes, yes, yes, buf, 1, s1, d1, buf, 0, s0, d0, next, 0);
    mask(2 * j - 1, s1);
    work(yes, yes, yes, next, 0, s0, d0, buf, 1, s1, d1, next, 1);
    advance();
  }
  mask(2 * nt - 2, s0);
  work(yes, yes, no, buf, 1, s1, d1, buf, 0, s0, d0, buf, 0);
  mask(2 * nt - 1, s1);
  work(no, yes, no, buf, 0, s0, d0, buf, 1, s1, d1, buf, 0);
  if (key < t.tokens) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4 x, y;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          x[jj] = (T)(ak[d][4 * i + jj] * a.scale);
          y[jj] = (T)av[d][4 * i + jj];
        }
        *reinterpret_cast<v4*>(dkr + (32 * d + 8 * i + 4 * h) * 2) = x;
        *reinterpret_cast<v4*>(dvr + (32 * d + 8 * i + 4 * h) * 2) = y;
      }
  }
}

template <typename T, int D>
static void launch_bwd(BwdArgs a, int64_t q_slots, int64_t k_slots, hipStream_t s) {
  a.slots = (int32_t)q_slots;
  hipLaunchKernelGGL((attn_bwd_dq_kernel<T, D>), dim3((unsigned)(q_slots * a.HKV)), dim3(256), 0, s, a);
  a.slots = (int32_t)k_slots;
  hipLaunchKernelGGL((attn_bwd_dkv_kernel<T, D>), dim3((unsigned)(k_slots * a.HKV)), dim3(256), 0, s, a);
}

}  // namespace attn
}  // namespace hmx

using namespace hmx;

extern "C" int hmx_causal_attention_bwd(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
    int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
    int64_t v_head_stride, int32_t dtype, const void* o, int64_t o_token_stride,
    int64_t o_head_stride, const void* dout, int64_t do_token_stride, int64_t do_head_stride,
    const float* lse, const int32_t* cu_seqlens, int32_t N, int64_t T, int32_t H, int32_t HKV,
    int32_t D, float scale, void* dq, int64_t dq_token_stride, int64_t dq_head_stride, void* dk,
    int64_t dk_token_stride, int64_t dk_head_stride, void* dv, int64_t dv_token_stride,
    int64_t dv_head_stride, float* delta, void* stream) {
  HMX_REQUIRE(D == 64 || D == 128, HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: head size %d not in {64, 128}", D);
  HMX_REQUIRE(dtype == HMX_BF16, HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: dtype code %d (bf16 only)", dtype);
  HMX_REQUIRE(N >= 0 && T >= 0 && HKV > 0 && H > 0 && H % HKV == 0, HMX_EINVAL,
              "hmx_causal_attention_bwd: N=%d T=%lld H=%d HKV=%d", N, (long long)T, H, HKV);
  HMX_REQUIRE(T * (H / HKV) < (1ll << 30), HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: %lld tokens",
              (long long)T);
  HMX_REQUIRE(scale > 0.f && scale < __builtin_inff(), HMX_EINVAL,
              "hmx_causal_attention_bwd: scale %g must be positive", (double)scale);
  HMX_REQUIRE(cu_seqlens || N == 0 || T % N == 0, HMX_EINVAL,
              "hmx_causal_attention_bwd: T=%lld is not N=%d sequences", (long long)T, N);
  if (T == 0 || (N == 0 && !cu_seqlens)) return HMX_OK;
  HMX_REQUIRE(q && k && v && o && dout && lse && dq && dk && dv && delta, HMX_EINVAL,
              "hmx_causal_attention_bwd: null pointer");
  const int64_t st = q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride |
                     v_head_stride | o_token_stride | o_head_stride | do_token_stride | do_head_stride |
                     dq_token_stride | dq_head_stride | dk_token_stride | dk_head_stride | dv_token_stride |
                     dv_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)dout |
                       (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0, HMX_EINVAL,
              "hmx_causal_attention_bwd: strides must be multiples of 8 elements and pointers 16-byte aligned");
  HMX_REQUIRE(attn::near_rows(k_token_stride) && attn::near_rows(v_token_stride), HMX_EUNSUPPORTED,
              "hmx_causal_attention_bwd: token strides of k and v past 2^25 elements");
  attn::BwdArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.o = (const char*)o;
  a.dout = (const char*)dout; a.dq = (char*)dq; a.dk = (char*)dk; a.dv = (char*)dv;
  a.q_ts = 2 * q_token_stride; a.q_hs = 2 * q_head_stride;
  a.k_ts = 2 * k_token_stride; a.k_hs = 2 * k_head_stride;
  a.v_ts = 2 * v_token_stride; a.v_hs = 2 * v_head_stride;
  a.o_ts = 2 * o_token_stride; a.o_hs = 2 * o_head_stride;
  a.do_ts = 2 * do_token_stride; a.do_hs = 2 * do_head_stride;
  a.dq_ts = 2 * dq_token_stride; a.dq_hs = 2 * dq_head_stride;
  a.dk_ts = 2 * dk_token_stride; a.dk_hs = 2 * dk_head_stride;
  a.dv_ts = 2 * dv_token_stride; a.dv_hs = 2 * dv_head_stride;
  a.lse = lse; a.delta = delta;
  a.seqs = attn::Seqs{cu_seqlens, N, (int32_t)T, H / HKV};
  a.G = attn::fast_div(H / HKV);
  a.H = H; a.HKV = HKV;
  a.c = scale * attn::LOG2E;
  a.scale = scale;
  const int64_t G = H / HKV, span = attn::KR / G;
  a.fixed = attn::KR % G == 0 && a.q_ts >= 0 && a.q_hs >= 0 && a.do_ts >= 0 && a.do_hs >= 0 && span * a.q_ts + G * a.q_hs < (1ll << 31) &&
            span * a.do_ts + G * a.do_hs < (1ll << 31);
  const int64_t qs = attn::tile_slots<attn::QM>(cu_seqlens, N, T, H / HKV);
  const int64_t ks = attn::tile_slots<attn::KM>(cu_seqlens, N, T, 1);
  HMX_REQUIRE(qs * HKV < (1ll << 31), HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: %lld tiles", (long long)qs);
  hipStream_t s = (hipStream_t)stream;
  if (D == 64) attn::launch_bwd<bf16, 64>(a, qs, ks, s);
  else attn::launch_bwd<bf16, 128>(a, qs, ks, s);
  return check_launch("hmx_causal_attention_bwd");
}
