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
// else stays in fp32.
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
  float* delta;        // [2, T, H]: delta, and lse - P_UP
  Seqs seqs;           // rows of tokens x G
  FastDiv G;
  int32_t H, HKV, slots;
  int32_t fixed;       // a tile's rows lie at fixed 32-bit offsets from its first token
  float c, scale;
};

constexpr int QM = 128;              // dQ: rows of a workgroup
constexpr float P_UP = 14.f;         // P is held times 2^14 for dK and dV: fp16 then keeps its precision down to 2^-28

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

  stage(0);
  for (int j = 0; j < nt; ++j) {
    const T *Kb = Ks[j & 1], *Vb = Vs[j & 1];
    dma_wait<0>();
    __syncthreads();
    if (j + 1 < nt) stage(j + 1);
    const int t0 = j * QN;
    if (t0 > w_last) continue;
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
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        ds[i] = __builtin_amdgcn_exp2f(st[i] * a.c - lse) * (dp[i] - delta);
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
  }
  // P sums to 1, so dS would sum to 0 had delta been formed from an exact O: what it does
  // sum to is delta's error, and dK gets a delta without it.
  over = pair_sum32(over, over);
  if (h == 0 && row < t.rows) {
    a.delta[gt * a.H + head] = delta + over;
    a.delta[((int64_t)a.seqs.T + gt) * a.H + head] = lse - P_UP;
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

constexpr int KM = 128, KR = 32;     // dK, dV: keys of a workgroup, rows of a unit

// Two waves share 32 keys and a SIMD: one forms S = Q K^T, P and dV^T += dO^T P, the other
// dP = dO V^T, dS and dK^T += Q^T dS, a unit of 32 rows behind; P goes from the first to the
// second through LDS in fp16 (2^-12 of it, against the 2^-9 of dS's own rounding).  The two
// are the same program over Q and dO in each other's places, and each holds one operand and
// one accumulator, so both fit a SIMD at 256 registers: where one wave did all of it, alone
// on its SIMD, its waits and its issue were the bound (2.69 ms at 8 x 4096 tokens, 32 / 8
// heads, against DKV_FIGURE).  In each, the next unit's first product is formed while this
// unit's exponentials (or differences) are.  Units arrive in LDS directly, in a ring of eight.
template <typename T, int D>
__global__ __launch_bounds__(512, 2) void attn_bwd_dkv_kernel(BwdArgs a) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int NC = D / 8, RI = 64 / NC, NL = 8 / RI, NS = D / 16, ND = D / 32;
  constexpr int RING = 8, UNIT = KR * D * 2;                 // bytes of a unit's Q, and of its dO
  __shared__ __align__(1024) char smem[RING * 2 * UNIT];     // [RING][Q, dO]
  __shared__ __align__(1024) f16 Ps[2][4][2][64][8];         // P of a unit: [unit][keys][half][lane]
  __shared__ __align__(16) float Ls[RING][2][KR];            // lse - 14 and delta of the rows

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = wave & 3, role = wave >> 2;
  const int kvh = blockIdx.x % a.HKV;
  Seqs sk = a.seqs;
  sk.G = 1;
  const Tile t = next_tile<KM, false>(sk, nullptr, blockIdx.x / a.HKV, a.slots);
  if (t.row0 >= t.rows || t.row0 < 0) return;
  const int key = t.row0 + grp * 32 + l32, keyc = min(key, t.tokens - 1);
  const int64_t gk = t.bos + keyc;
  char* out = role ? a.dk + gk * a.dk_ts + (int64_t)kvh * a.dk_hs : a.dv + gk * a.dv_ts + (int64_t)kvh * a.dv_hs;
  if (t.seq < 0) {
    if (key < t.tokens)
#pragma unroll
      for (int i = 0; i < NS; ++i) *reinterpret_cast<u32x4*>(out + 32 * i + 16 * h) = u32x4{0, 0, 0, 0};
    return;
  }
  v8 of[NS];                                // the wave's operand: its keys' K, or their V
  {
    const char* kv = role ? a.v + gk * a.v_ts + (int64_t)kvh * a.v_hs : a.k + gk * a.k_ts + (int64_t)kvh * a.k_hs;
#pragma unroll
    for (int s = 0; s < NS; ++s) of[s] = *reinterpret_cast<const v8*>(kv + 32 * s + 16 * h);
  }
  const int G = a.G.d, rows = t.tokens * G, nu = (rows + KR - 1) / KR;
  const int wk0 = min(t.row0 + grp * 32, t.tokens - 1);            // the wave's first key
  const int u_wg = t.row0 * G / KR, u_own = wk0 * G / KR;          // first units with rows that see them
  const int first = key * G;                                        // the key's first row

  // Staging: waves 0-3 bring Q's rows of a unit, 4-7 dO's, 8 each.  Where G divides a unit's
  // rows, a lane's rows of all units are one head's, at offsets that do not change.
  const int64_t r_ts = role ? a.do_ts : a.q_ts, r_hs = role ? a.do_hs : a.q_hs;
  const char* rbase = uniform_ptr((role ? a.dout : a.q) + (int64_t)t.bos * r_ts + (int64_t)kvh * G * r_hs);
  uint32_t roff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int x = grp * 8 + i * RI + lane / NC, tk = fdiv(x, a.G), g = x - tk * G;
    roff[i] = (uint32_t)(tk * r_ts + g * r_hs + 16 * swz<D>(x, lane % NC));
  }
  const int tpu = KR / G;                   // tokens of a unit where G divides it
  auto stage = [&](int u) __attribute__((always_inline)) {
    const int slot = u % RING;
    const uint32_t lds = lds_addr(smem) + (slot * 2 + role) * UNIT + grp * 8 * D * 2;
    if (a.fixed && (u + 1) * KR <= rows) {
      const char* b = uniform_ptr(rbase + (int64_t)u * tpu * r_ts);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(lds + i * RI * D * 2, b, roff[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int x = grp * 8 + i * RI + lane / NC, r = min(u * KR + x, rows - 1), tk = fdiv(r, a.G);
        dma16(lds + i * RI * D * 2, rbase + tk * r_ts + (r - tk * G) * r_hs + 16 * swz<D>(x, lane % NC));
      }
    }
    // the rows' terms, 32 lanes each (every wave brings them: its loads are counted)
    const int r = min(u * KR + l32, rows - 1), tk = fdiv(r, a.G);
    const float* terms = a.delta + (h ? 0 : (int64_t)a.seqs.T * a.H);
    dma4(lds_addr(&Ls[slot][0][0]),
         reinterpret_cast<const char*>(terms + ((int64_t)(t.bos + tk) * a.H + kvh * G + r - tk * G)));
  };
  int ro[NS], to[ND], tu[ND];               // byte offsets into a unit: rows, and columns of the other operand
#pragma unroll
  for (int s = 0; s < NS; ++s) ro[s] = role * UNIT + (l32 * D + swz<D>(l32, 2 * s + h) * 8) * 2;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    to[d] = (1 - role) * UNIT + tr_offset<D>(lane, d, false) * 2;
    tu[d] = (1 - role) * UNIT + tr_offset<D>(lane, d, true) * 2;
  }
  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x16{0};

  auto mask = [&](int u, f32x16& st) __attribute__((always_inline)) {
    // rows before the key do not see it, and rows behind the last are none
    if (u * KR < (wk0 + 31) * G || (u + 1) * KR > rows) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = u * KR + 8 * (i >> 2) + 4 * h + (i & 3);
        if (r < first || r >= rows) st[i] = NEG_INF;
      }
    }
  };
  // The first product of unit u + 1 into sn (NEXT), and what follows from unit u's, st (THIS).
  // LDS reads run AHEAD steps before their use.
  constexpr int AHEAD = 2, E = 16 / NS;
  auto work = [&](auto ROLE, auto NEXT, auto THIS, int u, f32x16& sn, const f32x16& st) __attribute__((always_inline)) {
    constexpr bool scores = decltype(ROLE)::value, next = decltype(NEXT)::value, cur = decltype(THIS)::value;
    const char *rn = smem + (u + 1) % RING * 2 * UNIT, *cc = smem + (u + RING) % RING * 2 * UNIT;
    v8 ra[NS], ct[2 * ND], pf[2];
    f32x4 term[4];
    f16x8 ph[2];
    float x[16];
    auto rows_of = [&](int s) __attribute__((always_inline)) { ra[s] = *reinterpret_cast<const v8*>(rn + ro[s]); };
    auto cols_of = [&](int g) __attribute__((always_inline)) {
      const char* c = cc + (g / ND) * 16 * D * 2;
      ct[g] = join<T>(tr4<T>(reinterpret_cast<const T*>(c + to[g % ND])), tr4<T>(reinterpret_cast<const T*>(c + tu[g % ND])));
    };
    if constexpr (next) {
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) rows_of(s);
    }
    if constexpr (cur) {
      const float* ls = &Ls[(u + RING) % RING][scores ? 0 : 1][4 * h];
#pragma unroll
      for (int i = 0; i < 4; ++i) term[i] = *reinterpret_cast<const f32x4*>(ls + 8 * i);
      if constexpr (!scores) {
#pragma unroll
        for (int b = 0; b < 2; ++b) ph[b] = *reinterpret_cast<const f16x8*>(&Ps[u & 1][grp][b][lane][0]);
      }
    }
    fence();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (next) {
        if (s + AHEAD < NS) rows_of(s + AHEAD);
      }
      if constexpr (cur) {
        if (s + AHEAD >= NS) cols_of(s + AHEAD - NS);
      }
      if constexpr (next) sn = El<T>::mma32(ra[s], of[s], s == 0 ? f32x16{0} : sn);
      if constexpr (cur) {
#pragma unroll
        for (int e = s * E; e < s * E + E; ++e)
          x[e] = scores ? __builtin_amdgcn_exp2f(st[e] * a.c - term[e >> 2][e & 3])
                        : (float)ph[e >> 3][e & 7] * (st[e] - term[e >> 2][e & 3]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
          if (s == (b + 1) * NS / 2 - 1) {
            const float* y = x + 8 * b;
            pf[b] = pack8<T>(y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]);
            if constexpr (scores)
              *reinterpret_cast<f16x8*>(&Ps[u & 1][grp][b][lane][0]) =
                  pack8<f16>(y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]);
          }
      }
      fence();
    }
    if constexpr (cur) {
#pragma unroll
      for (int g = 0; g < 2 * ND; ++g) {
        if (g + AHEAD < 2 * ND) cols_of(g + AHEAD);
        acc[g % ND] = El<T>::mma32(ct[g], pf[g / ND], acc[g % ND]);
        fence();
      }
    }
  };
  // step k: unit k + 1 is there, the RING - 3 after it on their way
  auto arrive = [&](int k) __attribute__((always_inline)) {
    if (k + RING - 3 < nu) dma_wait<(RING - 4) * (NL + 1)>();
    else dma_wait<0>();
    __syncthreads();
    if (k + RING - 2 < nu) stage(k + RING - 2);
  };
  // the first waves take unit k at step k, the others unit k - 1
  auto run = [&](auto ROLE) __attribute__((always_inline)) {
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    constexpr int lag = decltype(ROLE)::value ? 0 : 1;
    f32x16 s0, s1;
    int k = u_wg - 1;
    for (; k - lag < u_own - 1; ++k) arrive(k);        // rows before the wave's keys
    arrive(k);
    work(ROLE, yes, no, k - lag, s0, s0);
    int u = ++k - lag;                                 // scored: in s0
    for (; u + 2 < nu; u += 2) {
      arrive(k++);
      if constexpr (!lag) mask(u, s0);
      work(ROLE, yes, yes, u, s1, s0);
      arrive(k++);
      if constexpr (!lag) mask(u + 1, s1);
      work(ROLE, yes, yes, u + 1, s0, s1);
    }
    arrive(k++);
    if constexpr (!lag) mask(u, s0);
    if (u + 1 < nu) {
      work(ROLE, yes, yes, u, s1, s0);
      arrive(k++);
      if constexpr (!lag) mask(u + 1, s1);
      work(ROLE, no, yes, u + 1, s0, s1);
    } else {
      work(ROLE, no, yes, u, s1, s0);
    }
    for (; k <= nu; ++k) arrive(k);
  };
#pragma unroll
  for (int i = 0; i < RING - 3; ++i)
    if (u_wg + i < nu) stage(u_wg + i);
  if (role == 0) run(std::true_type{});
  else run(std::false_type{});
  if (key < t.tokens) {
    const float f = __builtin_amdgcn_exp2f(-P_UP) * (role ? a.scale : 1.f);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4 y;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) y[jj] = (T)(acc[d][4 * i + jj] * f);
        *reinterpret_cast<v4*>(out + (32 * d + 8 * i + 4 * h) * 2) = y;
      }
  }
}

template <typename T, int D>
static void launch_bwd(BwdArgs a, int64_t q_slots, int64_t k_slots, hipStream_t s) {
  a.slots = (int32_t)q_slots;
  hipLaunchKernelGGL((attn_bwd_dq_kernel<T, D>), dim3((unsigned)(q_slots * a.HKV)), dim3(256), 0, s, a);
  a.slots = (int32_t)k_slots;
  hipLaunchKernelGGL((attn_bwd_dkv_kernel<T, D>), dim3((unsigned)(k_slots * a.HKV)), dim3(512), 0, s, a);
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
  a.fixed = attn::KR % G == 0 && span * a.q_ts + G * a.q_hs < (1ll << 31) &&
            span * a.do_ts + G * a.do_hs < (1ll << 31);
  const int64_t qs = attn::tile_slots<attn::QM>(cu_seqlens, N, T, H / HKV);
  const int64_t ks = attn::tile_slots<attn::KM>(cu_seqlens, N, T, 1);
  HMX_REQUIRE(qs * HKV < (1ll << 31), HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: %lld tiles", (long long)qs);
  hipStream_t s = (hipStream_t)stream;
  if (D == 64) attn::launch_bwd<bf16, 64>(a, qs, ks, s);
  else attn::launch_bwd<bf16, 128>(a, qs, ks, s);
  return check_launch("hmx_causal_attention_bwd");
}
