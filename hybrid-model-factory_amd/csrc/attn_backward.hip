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
  float c, scale;
};

constexpr int QM = 128;              // dQ: rows of a workgroup

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void attn_bwd_dq_kernel(BwdArgs a) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int QN = D == 128 ? 32 : 64;    // keys of a tile
  constexpr int NC = D / 8, NL = QN * NC / 256, NS = D / 16, ND = D / 32;
  __shared__ __align__(16) T Ks[2][QN * D];
  __shared__ __align__(16) T Vs[2][QN * D];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, l32 = lane & 31;
  const int kvh = blockIdx.x % a.HKV;
  const Tile t = find_tile<QM>(a.seqs, a.slots - 1 - (int)(blockIdx.x / a.HKV));
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
  if (h == 0 && row < t.rows) a.delta[gt * a.H + head] = delta;

  const int srow = tid / NC, sc = tid % NC;
  constexpr int SR = 256 / NC;
  u32x4 kr[NL], vr[NL];
  auto load_tile = [&](int j) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int64_t r = t.bos + min(j * QN + srow + i * SR, keys - 1);
      kr[i] = *reinterpret_cast<const u32x4*>(a.k + r * a.k_ts + (int64_t)kvh * a.k_hs + 16 * sc);
      vr[i] = *reinterpret_cast<const u32x4*>(a.v + r * a.v_ts + (int64_t)kvh * a.v_hs + 16 * sc);
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

  load_tile(0);
  for (int j = 0; j < nt; ++j) {
    T *Kb = Ks[j & 1], *Vb = Vs[j & 1];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = srow + i * SR;
      *reinterpret_cast<u32x4*>(Kb + r * D + swz<D>(r, sc) * 8) = kr[i];
      *reinterpret_cast<u32x4*>(Vb + r * D + swz<D>(r, sc) * 8) = vr[i];
    }
    __syncthreads();
    if (j + 1 < nt) load_tile(j + 1);
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
      const bool masked = t0 + kt * 32 + 31 > w_first;
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float p = __builtin_amdgcn_exp2f(st[i] * a.c - lse);
        if (masked && t0 + kt * 32 + 8 * (i >> 2) + 4 * h + (i & 3) > tok) p = 0.f;
        ds[i] = p * (dp[i] - delta);
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

constexpr int KM = 128, KR = 32;     // dK, dV: keys of a workgroup, rows of a step

template <typename T, int D>
__global__ __launch_bounds__(256, 1) void attn_bwd_dkv_kernel(BwdArgs a) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int NC = D / 8, NL = KR * NC / 256, NS = D / 16, ND = D / 32;
  __shared__ __align__(16) T Qs[2][KR * D];
  __shared__ __align__(16) T Os[2][KR * D];
  __shared__ __align__(16) float Ls[2][2][KR];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, l32 = lane & 31;
  const int kvh = blockIdx.x % a.HKV;
  Seqs ks = a.seqs;
  ks.G = 1;
  const Tile t = find_tile<KM>(ks, (int)(blockIdx.x / a.HKV));
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
  const int rows = t.tokens * a.G.d;
  const int j0 = (int)((int64_t)t.row0 * a.G.d / KR), nt = (rows + KR - 1) / KR;
  const int wk0 = t.row0 + wave * 32;       // the wave's first key

  const int srow = tid / NC, sc = tid % NC;
  constexpr int SR = 256 / NC;
  u32x4 qr[NL], dr[NL];
  float lr = 0.f;
  auto load_tile = [&](int j) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = min(j * KR + srow + i * SR, rows - 1), tk = fdiv(r, a.G);
      const int64_t hd = kvh * a.G.d + r - tk * a.G.d, g = t.bos + tk;
      qr[i] = *reinterpret_cast<const u32x4*>(a.q + g * a.q_ts + hd * a.q_hs + 16 * sc);
      dr[i] = *reinterpret_cast<const u32x4*>(a.dout + g * a.do_ts + hd * a.do_hs + 16 * sc);
    }
    if (tid < 2 * KR) {
      const int r0 = j * KR + (tid & (KR - 1)), r = min(r0, rows - 1), tk = fdiv(r, a.G);
      const int64_t at = (int64_t)(t.bos + tk) * a.H + kvh * a.G.d + r - tk * a.G.d;
      lr = (tid < KR ? a.lse : a.delta)[at];
      if (tid < KR && r0 >= rows) lr = __builtin_inff();   // no row: its P is 0
    }
  };
  int qo[NS], to[ND], tu[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s) qo[s] = l32 * D + swz<D>(l32, 2 * s + h) * 8;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    to[d] = tr_offset<D>(lane, d, false);
    tu[d] = tr_offset<D>(lane, d, true);
  }
  f32x16 ak[ND], av[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) ak[i] = av[i] = f32x16{0};

  load_tile(j0);
  for (int j = j0; j < nt; ++j) {
    T *Qb = Qs[j & 1], *Ob = Os[j & 1];
    float* Lb = &Ls[j & 1][0][0];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = srow + i * SR;
      *reinterpret_cast<u32x4*>(Qb + r * D + swz<D>(r, sc) * 8) = qr[i];
      *reinterpret_cast<u32x4*>(Ob + r * D + swz<D>(r, sc) * 8) = dr[i];
    }
    if (tid < 2 * KR) Lb[tid] = lr;
    __syncthreads();
    if (j + 1 < nt) load_tile(j + 1);
    const int r_last = min(j * KR + KR, rows) - 1;
    if (fdiv(r_last, a.G) < wk0) continue;  // every row of the step lies before the wave's keys
    const bool masked = fdiv(j * KR, a.G) < wk0 + 31;

    f32x16 st = {0}, dp = {0};
#pragma unroll
    for (int s = 0; s < NS; ++s) st = El<T>::mma32(*reinterpret_cast<const v8*>(Qb + qo[s]), kf[s], st);
#pragma unroll
    for (int s = 0; s < NS; ++s) dp = El<T>::mma32(*reinterpret_cast<const v8*>(Ob + qo[s]), vf[s], dp);
    float p[16], ds[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 ls = *reinterpret_cast<const f32x4*>(Lb + 8 * i + 4 * h);
      const f32x4 dl = *reinterpret_cast<const f32x4*>(Lb + KR + 8 * i + 4 * h);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int e = 4 * i + x;
        p[e] = __builtin_amdgcn_exp2f(st[e] * a.c - ls[x]);
        if (masked && fdiv(min(j * KR + 8 * i + 4 * h + x, rows - 1), a.G) < key) p[e] = 0.f;
        ds[e] = p[e] * (dp[e] - dl[x]);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int b = 8 * s;
      const v8 pf = pack8<T>(p[b], p[b + 1], p[b + 2], p[b + 3], p[b + 4], p[b + 5], p[b + 6], p[b + 7]);
      const v8 sf = pack8<T>(ds[b], ds[b + 1], ds[b + 2], ds[b + 3], ds[b + 4], ds[b + 5], ds[b + 6], ds[b + 7]);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const T *op = Ob + s * 16 * D, *qp = Qb + s * 16 * D;
        av[d] = El<T>::mma32(join<T>(tr4<T>(op + to[d]), tr4<T>(op + tu[d])), pf, av[d]);
        ak[d] = El<T>::mma32(join<T>(tr4<T>(qp + to[d]), tr4<T>(qp + tu[d])), sf, ak[d]);
      }
    }
  }
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
  HMX_REQUIRE(T * (H / HKV) < (1ll << 31) - 256, HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: %lld tokens",
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
  const int64_t qs = attn::tile_slots<attn::QM>(cu_seqlens, N, T, H / HKV);
  const int64_t ks = attn::tile_slots<attn::KM>(cu_seqlens, N, T, 1);
  HMX_REQUIRE(qs * HKV < (1ll << 31), HMX_EUNSUPPORTED, "hmx_causal_attention_bwd: %lld tiles", (long long)qs);
  hipStream_t s = (hipStream_t)stream;
  if (D == 64) attn::launch_bwd<bf16, 64>(a, qs, ks, s);
  else attn::launch_bwd<bf16, 128>(a, qs, ks, s);
  return check_launch("hmx_causal_attention_bwd");
}
