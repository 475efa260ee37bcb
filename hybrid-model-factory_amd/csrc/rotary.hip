// The position rotation of q and k by frequencies, and its gradient's:
//   (x1, x2) -> f (x1 cos a - x2 sin a, x2 cos a + x1 sin a),  a = position * inv_freq[i]
// for the pairs (i, i + R/2) or (2i, 2i + 1) of the first R elements of every head; the others
// are copied.  The gradient turns by -a.  fp32 arithmetic, one rounding; the angle is formed in
// 64 bits and taken modulo a turn there: at position 2^20 an fp32 product would be off by 2^-4.
//
// Layout: as where the cache is filled (paged_kv.hip) a thread owns two 8-element chunks of a
// head that hold whole pairs, forms its eight angles once and walks `per` heads of its token
// with their cosines and sines in registers, BATCH heads' loads ahead of their stores.
// Bound by memory: q and k in and out.  Measured: 8 x 4096 tokens, 32 / 8 heads of 128, 136 us,
// 4.9 TB/s, what a large copy reaches; 100003 tokens of 16 / 4 heads, half of each turned,
// 189 us, 5.4 TB/s; 197 tokens 5 us, a launch.
#include "attn.hpp"

namespace hmx {
namespace rotary {

struct Tensor {
  const char* in;
  char* out;
  int64_t bs, ts, hs, obs, ots, ohs;      // bytes
};
struct Args {
  Tensor q, k;
  const void *pos, *inv;
  int64_t pos_stride;
  attn::FastDiv T;
  float factor;
  int32_t pos64, inv64, R, inter, back, tokens, H, HKV, per;
};

// cos and sin of a position's angle, times the factor
__device__ __forceinline__ void turn_of(double pos, double inv, float factor, float& c, float& s) {
  const double t = pos * inv * 0.15915494309189535;   // turns
  float sn, cs;
  sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
  c = cs * factor;
  s = sn * factor;
}
__device__ __forceinline__ double freq_at(const void* p, int i, int is64) {
  return is64 ? static_cast<const double*>(p)[i] : (double)static_cast<const float*>(p)[i];
}

template <typename V, bool FAR> __device__ __forceinline__ V load16(const char* p) {
  typedef attn::u32x4 u;
  if constexpr (FAR) return __builtin_bit_cast(V, __builtin_nontemporal_load(reinterpret_cast<const u*>(p)));
  else return *reinterpret_cast<const V*>(p);
}
template <bool FAR, typename V> __device__ __forceinline__ void store16(char* p, V x) {
  typedef attn::u32x4 u;
  if constexpr (FAR) __builtin_nontemporal_store(__builtin_bit_cast(u, x), reinterpret_cast<u*>(p));
  else *reinterpret_cast<V*>(p) = x;
}

// FAR: past the caches' allocation, where q and k in and out are more than they hold (100003
// tokens, 16 / 4 heads of 128: 202 -> 189 us; 8192 such tokens, which they hold, 18.2 -> 20.9).
template <typename T, int D, bool FAR>
__global__ __launch_bounds__(256) void rotary_kernel(Args a) {
  typedef typename attn::El<T>::v8 v8;
  constexpr int TPR = D / 16;             // threads of a row
  constexpr int TPB = 256 / TPR;          // tokens of a workgroup
  constexpr int BATCH = 4;
  const int j = threadIdx.x % TPR;
  const int n = blockIdx.x * TPB + threadIdx.x / TPR;
  if (n >= a.tokens) return;
  const int b = attn::fdiv(n, a.T);
  const int64_t t = n - (int64_t)b * a.T.d;
  // Halves pair chunk j with j + rc; chunks that hold whole pairs, and those that do not
  // rotate, are paired so that a row's lanes read and write neighbouring chunks.
  const int rc = a.R >> 4;
  const int c0 = a.inter || j < rc ? j : 2 * rc + j - rc, c1 = a.inter ? j + TPR : j < rc ? j + rc : c0 + TPR - rc;
  const bool rot0 = a.inter ? c0 < 2 * rc : j < rc, rot1 = a.inter ? c1 < 2 * rc : j < rc;
  float cs[8], sn[8];
  if (rot0) {
    const int64_t at = b * a.pos_stride + t;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at] : (double)static_cast<const int32_t*>(a.pos)[at];
    // halves: pair 8 j + i of the head; neighbours: pairs 4 c .. 4 c + 3 of either chunk
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (a.inter && i >= 4 && !rot1) break;
      const int pair = a.inter ? 4 * (i < 4 ? c0 : c1) + (i & 3) : 8 * j + i;
      turn_of(pos, freq_at(a.inv, pair, a.inv64), a.factor, cs[i], sn[i]);
      if (a.back) sn[i] = -sn[i];
    }
  }
  const int h1 = min(a.H + a.HKV, (int)(blockIdx.y + 1) * a.per);
  for (int h0 = blockIdx.y * a.per; h0 < h1; h0 += BATCH) {
    v8 x[BATCH], y[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = min(h0 + i, h1 - 1);
      const char* p = h < a.H ? a.q.in + b * a.q.bs + t * a.q.ts + h * a.q.hs
                              : a.k.in + b * a.k.bs + t * a.k.ts + (h - a.H) * a.k.hs;
      x[i] = load16<v8, FAR>(p + 16 * c0);
      y[i] = load16<v8, FAR>(p + 16 * c1);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i;
      if (h >= h1) break;
      if (rot0) {
        float u[8], w[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          u[z] = (float)x[i][z];
          w[z] = (float)y[i][z];
        }
        if (a.inter) {
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            x[i][2 * z] = (T)(u[2 * z] * cs[z] - u[2 * z + 1] * sn[z]);
            x[i][2 * z + 1] = (T)(u[2 * z + 1] * cs[z] + u[2 * z] * sn[z]);
            if (!rot1) continue;
            y[i][2 * z] = (T)(w[2 * z] * cs[4 + z] - w[2 * z + 1] * sn[4 + z]);
            y[i][2 * z + 1] = (T)(w[2 * z + 1] * cs[4 + z] + w[2 * z] * sn[4 + z]);
          }
        } else {
#pragma unroll
          for (int z = 0; z < 8; ++z) {
            x[i][z] = (T)(u[z] * cs[z] - w[z] * sn[z]);
            y[i][z] = (T)(w[z] * cs[z] + u[z] * sn[z]);
          }
        }
      }
      char* p = h < a.H ? a.q.out + b * a.q.obs + t * a.q.ots + h * a.q.ohs
                        : a.k.out + b * a.k.obs + t * a.k.ots + (h - a.H) * a.k.ohs;
      store16<FAR>(p + 16 * c0, x[i]);
      store16<FAR>(p + 16 * c1, y[i]);
    }
  }
}

template <typename T, int D>
static void launch(const Args& a, bool far, dim3 grid, hipStream_t s) {
  if (far) hipLaunchKernelGGL((rotary_kernel<T, D, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, D, false>), grid, dim3(256), 0, s, a);
}

__global__ __launch_bounds__(256) void table_kernel(const void* inv, int inv64, float factor, int64_t positions, int R,
                                                    float* table) {
  const int half = R >> 1;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < positions * half; at += (int64_t)gridDim.x * 256) {
    const int64_t p = at / half;
    const int i = (int)(at - p * half);
    turn_of((double)p, freq_at(inv, i, inv64), factor, table[p * R + i], table[p * R + half + i]);
  }
}

}  // namespace rotary
}  // namespace hmx

using namespace hmx;

extern "C" int hmx_rotary_embedding(const void* q, int64_t q_batch_stride, int64_t q_token_stride,
                                    int64_t q_head_stride, void* q_out, int64_t q_out_batch_stride,
                                    int64_t q_out_token_stride, int64_t q_out_head_stride, const void* k,
                                    int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                                    void* k_out, int64_t k_out_batch_stride, int64_t k_out_token_stride,
                                    int64_t k_out_head_stride, int32_t dtype, const void* positions,
                                    int32_t positions_int64, int64_t positions_stride, const void* inv_freq,
                                    int32_t inv_freq_f64, float factor, int32_t rotary_dim,
                                    int32_t interleaved, int32_t backward, int32_t B, int64_t T, int32_t H,
                                    int32_t HKV, int32_t D, void* stream) {
  HMX_REQUIRE(D == 64 || D == 128, HMX_EUNSUPPORTED, "hmx_rotary_embedding: head size %d not in {64, 128}", D);
  HMX_REQUIRE(dtype == HMX_BF16 || dtype == HMX_F16, HMX_EUNSUPPORTED,
              "hmx_rotary_embedding: dtype code %d (bf16 or fp16)", dtype);
  HMX_REQUIRE(rotary_dim > 0 && rotary_dim <= D && rotary_dim % 16 == 0, HMX_EUNSUPPORTED,
              "hmx_rotary_embedding: rotary_dim %d (a multiple of 16 up to the head size)", rotary_dim);
  HMX_REQUIRE(B >= 0 && T >= 0 && H > 0 && HKV >= 0 && (k || HKV == 0), HMX_EINVAL,
              "hmx_rotary_embedding: B=%d T=%lld heads %d / %d", B, (long long)T, H, HKV);
  if (B == 0 || T == 0) return HMX_OK;
  HMX_REQUIRE(T < (1ll << 31) && B * T < (1ll << 31) - 256, HMX_EUNSUPPORTED, "hmx_rotary_embedding: %d x %lld tokens", B,
              (long long)T);
  HMX_REQUIRE(q && q_out && (HKV == 0 || k_out) && positions && inv_freq, HMX_EINVAL,
              "hmx_rotary_embedding: null pointer");
  const int64_t st = q_batch_stride | q_token_stride | q_head_stride | q_out_batch_stride | q_out_token_stride |
                     q_out_head_stride | k_batch_stride | k_token_stride | k_head_stride | k_out_batch_stride |
                     k_out_token_stride | k_out_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0, HMX_EINVAL,
              "hmx_rotary_embedding: strides must be multiples of 8 elements and pointers 16-byte aligned");
  rotary::Args a{};
  a.q = rotary::Tensor{(const char*)q, (char*)q_out, 2 * q_batch_stride, 2 * q_token_stride, 2 * q_head_stride,
                       2 * q_out_batch_stride, 2 * q_out_token_stride, 2 * q_out_head_stride};
  a.k = rotary::Tensor{(const char*)k, (char*)k_out, 2 * k_batch_stride, 2 * k_token_stride, 2 * k_head_stride,
                       2 * k_out_batch_stride, 2 * k_out_token_stride, 2 * k_out_head_stride};
  a.pos = positions; a.pos64 = positions_int64; a.pos_stride = positions_stride;
  a.inv = inv_freq; a.inv64 = inv_freq_f64; a.factor = factor;
  a.T = attn::fast_div((int32_t)T);
  a.R = rotary_dim; a.inter = interleaved; a.back = backward;
  a.tokens = (int32_t)(B * T); a.H = H; a.HKV = HKV;
  const int heads = H + HKV, tpb = 256 / (D / 16);
  const int64_t bx = ((int64_t)a.tokens + tpb - 1) / tpb;
  // heads of a thread: as many as leave eight workgroups a compute unit, in whole batches
  const int64_t want = 8ll * cu_count(), by = bx >= want ? 1 : (want + bx - 1) / bx;
  a.per = (int)((heads + by - 1) / by);
  a.per = (a.per + 3) / 4 * 4;
  const dim3 grid((unsigned)bx, (unsigned)((heads + a.per - 1) / a.per));
  hipStream_t s = (hipStream_t)stream;
  const bool far = 4ll * a.tokens * heads * D > 256ll << 20;   // of the last cache's 256 MB
  if (dtype == HMX_BF16) {
    if (D == 64) rotary::launch<bf16, 64>(a, far, grid, s);
    else rotary::launch<bf16, 128>(a, far, grid, s);
  } else {
    if (D == 64) rotary::launch<f16, 64>(a, far, grid, s);
    else rotary::launch<f16, 128>(a, far, grid, s);
  }
  return check_launch("hmx_rotary_embedding");
}

extern "C" int hmx_rotary_table(const void* inv_freq, int32_t inv_freq_f64, float factor, int64_t positions,
                                int32_t rotary_dim, float* table, void* stream) {
  HMX_REQUIRE(positions >= 0 && rotary_dim > 0 && rotary_dim % 2 == 0, HMX_EINVAL,
              "hmx_rotary_table: %lld positions of %d", (long long)positions, rotary_dim);
  if (positions == 0) return HMX_OK;
  HMX_REQUIRE(inv_freq && table, HMX_EINVAL, "hmx_rotary_table: null pointer");
  const int64_t blocks = (positions * (rotary_dim / 2) + 255) / 256, most = 16ll * cu_count();
  hipLaunchKernelGGL(rotary::table_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0,
                     (hipStream_t)stream, inv_freq, inv_freq_f64, factor, positions, rotary_dim, table);
  return check_launch("hmx_rotary_table");
}
