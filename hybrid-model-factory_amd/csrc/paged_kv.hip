// Appending keys and values to a paged cache, with the position rotation of q and k:
//   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin),  cos, sin = table[position]
// for the pairs (i, i + R/2) or (2i, 2i + 1) of the first R elements of every head; the
// others and v are copied.  fp32 arithmetic, one rounding.
//
// Layout: a thread owns two 8-element chunks of a head that hold whole pairs (chunks j
// and j + R/16 for halves), so a pair never crosses lanes, and walks `per` heads of one
// token with its cos and sin in registers.  Bound by memory: q in and out, k and v in and
// out, one table row a token; few tokens are bound by the launch, so then a thread takes
// one head (`per` = 1) and the heads spread over workgroups.  Measured, 32 / 8 heads of 128:
// 30011 tokens 154 us, 4.8 TB/s, what a large copy reaches; 8 tokens 19 us a call, the launch
// and its host work.
//
// A cache of 8 bits (Q8): the row's largest magnitude, joined over the D / 16 lanes that hold
// it, gives its power of two, and the row goes out as e4m3 with one byte of scale.  Measured, 30011
// tokens 144 us, 4.8 TB/s; 8 tokens 4.1, and 18 a call.
#include "attn.hpp"

namespace hmx {
namespace pkv {

struct Args {
  const void *q, *k, *v;
  void* qo;
  void *kc, *vc;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs;
  int64_t k_ps, k_cts, k_chs, v_ps, v_cts, v_chs;
  const void *slots, *pos, *cs;
  int64_t cs_stride, max_pos, num_slots;
  int32_t slots64, pos64, cs_dt, R, inter, tokens, H, HKV, per, eight;
  attn::FastDiv page;
  uint8_t *k_sc, *v_sc;                   // bytes of scale, of a cache of 8 bits
  int64_t k_sc_ps, k_sc_hs, v_sc_ps, v_sc_hs;
};

__device__ __forceinline__ int64_t index_at(const void* p, int i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

template <typename C>
__device__ __forceinline__ void load_cs(const C* p, int R, float* cs, float* sn) {
  load_vec<8>(p, cs);
  load_vec<8>(p + (R >> 1), sn);
}

// The thread's pairs turned, each product and each sum rounded by itself: what is stored in 8
// bits is then the same for everybody who forms it by these operations (a contracted product
// moves a value across a border of e4m3 now and then, and a row's largest across a scale's).
__device__ __forceinline__ void turn_exact(float* x, float* y, const float* cs, const float* sn, bool inter) {
#pragma clang fp contract(off)
  if (inter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x1 = x[2 * i], x2 = x[2 * i + 1], y1 = y[2 * i], y2 = y[2 * i + 1];
      x[2 * i] = x1 * cs[i] - x2 * sn[i];
      x[2 * i + 1] = x2 * cs[i] + x1 * sn[i];
      y[2 * i] = y1 * cs[4 + i] - y2 * sn[4 + i];
      y[2 * i + 1] = y2 * cs[4 + i] + y1 * sn[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x1 = x[i], x2 = y[i];
      x[i] = x1 * cs[i] - x2 * sn[i];
      y[i] = x2 * cs[i] + x1 * sn[i];
    }
  }
}

// The byte of scale of a row whose largest finite magnitude is m: 2^(code - 127) is the least
// power of two, from 2^-126 on, of which m is at most 448 = 1.75 * 2^8.  A power of two costs
// e4m3 nothing (its steps are relative) but one binary order of range below, and both ways of
// it are exact.
__device__ __forceinline__ uint32_t scale_code(float m) {
  const uint32_t b = __builtin_bit_cast(uint32_t, m);
  return (uint32_t)max((int)(b >> 23) - 8 + ((b & 0x7fffff) > 0x600000 ? 1 : 0), 1);
}
// Eight values times inv in e4m3, to the nearest, ties to even; what is not finite becomes NaN.
__device__ __forceinline__ attn::u32x2 to_e4m3(const float* x, float inv) {
  attn::u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const float v = x[4 * i + z];
      y[z] = __builtin_fabsf(v) < __builtin_inff() ? v * inv : __builtin_nanf("");
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    r[i] = (uint32_t)w;
  }
  return r;
}

template <typename T, int D, bool Q8>
__global__ __launch_bounds__(256) void append_kernel(Args a) {
  constexpr int TPR = D / 16;             // threads of a row
  constexpr int TPB = 256 / TPR;          // tokens of a workgroup
  const int j = threadIdx.x % TPR;
  const int t = blockIdx.x * TPB + threadIdx.x / TPR;
  if (t >= a.tokens) return;
  const int rc = a.R >> 4;                // chunk pairs that rotate
  const bool rot = j < rc;
  // the thread's two chunks: halves pair chunk j with j + rc; what does not rotate, and
  // pairs inside a chunk, take neighbours
  const int c0 = rot ? (a.inter ? 2 * j : j) : 2 * j;
  const int c1 = rot && !a.inter ? j + rc : c0 + 1;
  float cs[8], sn[8];
  if (rot) {
    const int64_t p = index_at(a.pos, t, a.pos64);
    const bool in = p >= 0 && p < a.max_pos;
    // pair i of the chunks: table column 8j + i for halves; for neighbours chunk c0 holds
    // pairs 8j..8j+3 and chunk c1 8j+4..8j+7: column 8j + i either way
    const int64_t row = (in ? p : 0) * a.cs_stride + 8 * j;
    if (a.cs_dt == HMX_F32) load_cs(static_cast<const float*>(a.cs) + row, a.R, cs, sn);
    else if (a.cs_dt == HMX_BF16) load_cs(static_cast<const bf16*>(a.cs) + row, a.R, cs, sn);
    else load_cs(static_cast<const f16*>(a.cs) + row, a.R, cs, sn);
    if (!in) {                            // a position outside the table
#pragma unroll
      for (int i = 0; i < 8; ++i) cs[i] = sn[i] = __builtin_nanf("");
    }
  }
  const int64_t slot = index_at(a.slots, t, a.slots64);
  const bool keep = slot >= 0 && slot < a.num_slots;
  const int64_t pg = keep ? attn::fdiv64(slot, a.page) : 0, at = keep ? slot - pg * a.page.d : 0;
  const int Hq = a.qo ? a.H : 0;
  const int h1 = min(Hq + 2 * a.HKV, (int)(blockIdx.y + 1) * a.per);
  for (int h = blockIdx.y * a.per; h < h1; ++h) {
    const bool is_q = h < Hq, is_v = h >= Hq + a.HKV;
    const int hh = is_q ? h : is_v ? h - Hq - a.HKV : h - Hq;
    if (!is_q && !keep) continue;
    const T* src = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) +
                   (int64_t)t * (is_q ? a.q_ts : is_v ? a.v_ts : a.k_ts) +
                   (int64_t)hh * (is_q ? a.q_hs : is_v ? a.v_hs : a.k_hs);
    const int64_t to = is_q ? (int64_t)t * a.qo_ts + (int64_t)hh * a.qo_hs
                            : is_v ? pg * a.v_ps + at * a.v_cts + hh * a.v_chs
                                   : pg * a.k_ps + at * a.k_cts + hh * a.k_chs;
    float x[8], y[8];
    load_vec<8>(src + 8 * c0, x);
    load_vec<8>(src + 8 * c1, y);
    if (Q8 && !is_q) {
      if (rot && !is_v) turn_exact(x, y, cs, sn, a.inter);
      float m = 0.f;                      // the row's largest finite magnitude, over its TPR lanes
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = __builtin_fabsf(x[i]), w = __builtin_fabsf(y[i]);
        m = fmaxf(m, u < __builtin_inff() ? u : 0.f);
        m = fmaxf(m, w < __builtin_inff() ? w : 0.f);
      }
#pragma unroll
      for (int z = 1; z < TPR; z <<= 1) m = fmaxf(m, __shfl_xor(m, z, 64));
      const uint32_t code = scale_code(m);
      const float inv = __builtin_bit_cast(float, (254 - code) << 23);
      uint8_t* dst = static_cast<uint8_t*>(is_v ? a.vc : a.kc) + to;
      *reinterpret_cast<attn::u32x2*>(dst + 8 * c0) = to_e4m3(x, inv);
      *reinterpret_cast<attn::u32x2*>(dst + 8 * c1) = to_e4m3(y, inv);
      if (j == 0) {
        if (is_v) a.v_sc[pg * a.v_sc_ps + hh * a.v_sc_hs + at] = (uint8_t)code;
        else a.k_sc[pg * a.k_sc_ps + hh * a.k_sc_hs + at] = (uint8_t)code;
      }
      continue;
    }
    if (rot && !is_v) {
      if (a.inter) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x1 = x[2 * i], x2 = x[2 * i + 1], y1 = y[2 * i], y2 = y[2 * i + 1];
          x[2 * i] = x1 * cs[i] - x2 * sn[i];
          x[2 * i + 1] = x2 * cs[i] + x1 * sn[i];
          y[2 * i] = y1 * cs[4 + i] - y2 * sn[4 + i];
          y[2 * i + 1] = y2 * cs[4 + i] + y1 * sn[4 + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x1 = x[i], x2 = y[i];
          x[i] = x1 * cs[i] - x2 * sn[i];
          y[i] = x2 * cs[i] + x1 * sn[i];
        }
      }
    }
    T* dst = static_cast<T*>(is_q ? a.qo : is_v ? a.vc : a.kc) + to;
    store_vec<8>(dst + 8 * c0, x);
    store_vec<8>(dst + 8 * c1, y);
  }
}

template <typename T, int D>
static void launch(const Args& a, dim3 grid, hipStream_t s) {
  if (a.eight) hipLaunchKernelGGL((append_kernel<T, D, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((append_kernel<T, D, false>), grid, dim3(256), 0, s, a);
}

}  // namespace pkv
}  // namespace hmx

using namespace hmx;

static int append_paged_kv(const char* what, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                           const void* k, int64_t k_token_stride, int64_t k_head_stride,
                           const void* v, int64_t v_token_stride, int64_t v_head_stride,
                           int32_t dtype, void* q_out, int64_t q_out_token_stride,
                           int64_t q_out_head_stride, const hmx_paged_kv* cache, const hmx_kv_scales* scales,
                           const void* slots, int32_t slots_int64, const void* positions,
                           int32_t positions_int64, const void* cos_sin,
                           int32_t cos_sin_dtype, int64_t cos_sin_stride,
                           int64_t max_position, int32_t rotary_dim, int32_t interleaved,
                           int64_t tokens, int32_t H, int32_t HKV, int32_t D, void* stream) {
  HMX_REQUIRE(D == 64 || D == 128, HMX_EUNSUPPORTED,
              "%s: head size %d not in {64, 128}", what, D);
  HMX_REQUIRE(dtype == HMX_BF16 || dtype == HMX_F16, HMX_EUNSUPPORTED,
              "%s: dtype code %d (bf16 or fp16)", what, dtype);
  HMX_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && H >= 0 && HKV > 0 && cache, HMX_EINVAL,
              "%s: tokens %lld, heads %d / %d", what, (long long)tokens, H, HKV);
  HMX_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0, HMX_EUNSUPPORTED,
              "%s: rotary_dim %d (a multiple of 16 up to the head size)", what, rotary_dim);
  HMX_REQUIRE(cache->num_pages >= 0 && cache->page_size > 0, HMX_EINVAL,
              "%s: %d pages of %d", what, cache->num_pages, cache->page_size);
  if (tokens == 0) return HMX_OK;
  HMX_REQUIRE(k && v && slots && (cache->num_pages == 0 || (cache->k && cache->v)) && (!q_out || q), HMX_EINVAL,
              "%s: null pointer", what);
  HMX_REQUIRE(rotary_dim == 0 || (positions && cos_sin && max_position > 0 &&
                                  cos_sin_dtype >= 0 && cos_sin_dtype <= 2),
              HMX_EINVAL, "%s: a rotation needs positions and their table", what);
  HMX_REQUIRE(rotary_dim == 0 || (cos_sin_stride % 8 == 0 && (uintptr_t)cos_sin % 16 == 0), HMX_EINVAL,
              "%s: the table's rows must be multiples of 8 elements, 16-byte aligned", what);
  const int64_t st = q_token_stride | q_head_stride | k_token_stride | k_head_stride |
                     v_token_stride | v_head_stride | q_out_token_stride | q_out_head_stride |
                     cache->k_page_stride | cache->k_token_stride | cache->k_head_stride |
                     cache->v_page_stride | cache->v_token_stride | cache->v_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out |
                       (uintptr_t)cache->k | (uintptr_t)cache->v;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0 && attn::aligned_pages(*cache, scales != nullptr), HMX_EINVAL,
              "%s: strides must be multiples of 8 elements (a cache's of 16 bytes) and pointers 16-byte aligned", what);
  HMX_REQUIRE(!scales || cache->num_pages == 0 || (scales->k && scales->v), HMX_EINVAL, "%s: null pointer", what);
  pkv::Args a{};
  a.q = q; a.k = k; a.v = v; a.qo = q_out; a.kc = cache->k; a.vc = cache->v;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride; a.k_ts = k_token_stride; a.k_hs = k_head_stride;
  a.v_ts = v_token_stride; a.v_hs = v_head_stride;
  a.qo_ts = q_out_token_stride; a.qo_hs = q_out_head_stride;
  a.k_ps = cache->k_page_stride; a.k_cts = cache->k_token_stride; a.k_chs = cache->k_head_stride;
  a.v_ps = cache->v_page_stride; a.v_cts = cache->v_token_stride; a.v_chs = cache->v_head_stride;
  a.slots = slots; a.pos = positions; a.cs = cos_sin;
  a.cs_stride = cos_sin_stride; a.max_pos = max_position;
  a.num_slots = (int64_t)cache->num_pages * cache->page_size;
  a.slots64 = slots_int64; a.pos64 = positions_int64; a.cs_dt = cos_sin_dtype;
  a.R = rotary_dim; a.inter = interleaved; a.tokens = (int32_t)tokens; a.H = H; a.HKV = HKV;
  a.page = attn::fast_div(cache->page_size);
  if (scales) {
    a.eight = 1;
    a.k_sc = scales->k; a.k_sc_ps = scales->k_page_stride; a.k_sc_hs = scales->k_head_stride;
    a.v_sc = scales->v; a.v_sc_ps = scales->v_page_stride; a.v_sc_hs = scales->v_head_stride;
  }
  const int heads = (q_out ? H : 0) + 2 * HKV;
  const int tpb = 256 / (D / 16);
  const int64_t bx = (tokens + tpb - 1) / tpb;
  // heads of a thread: as many as leave four workgroups a CU, so that few tokens still
  // fill the chip and many read their table rows once
  const int64_t want = 4ll * cu_count();
  const int64_t by = bx >= want ? 1 : (want + bx - 1) / bx;
  a.per = (int)((heads + by - 1) / by);
  if (a.per > 8) a.per = 8;
  const dim3 grid((unsigned)bx, (unsigned)((heads + a.per - 1) / a.per));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == HMX_BF16) {
    if (D == 64) pkv::launch<bf16, 64>(a, grid, s);
    else pkv::launch<bf16, 128>(a, grid, s);
  } else {
    if (D == 64) pkv::launch<f16, 64>(a, grid, s);
    else pkv::launch<f16, 128>(a, grid, s);
  }
  return check_launch(what);
}

extern "C" int hmx_append_paged_kv(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                   const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                   const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                   int32_t dtype, void* q_out, int64_t q_out_token_stride,
                                   int64_t q_out_head_stride, const hmx_paged_kv* cache,
                                   const void* slots, int32_t slots_int64, const void* positions,
                                   int32_t positions_int64, const void* cos_sin,
                                   int32_t cos_sin_dtype, int64_t cos_sin_stride,
                                   int64_t max_position, int32_t rotary_dim, int32_t interleaved,
                                   int64_t tokens, int32_t H, int32_t HKV, int32_t D,
                                   void* stream) {
  return append_paged_kv("hmx_append_paged_kv", q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v,
                         v_token_stride, v_head_stride, dtype, q_out, q_out_token_stride, q_out_head_stride, cache,
                         nullptr, slots, slots_int64, positions, positions_int64, cos_sin, cos_sin_dtype,
                         cos_sin_stride, max_position, rotary_dim, interleaved, tokens, H, HKV, D, stream);
}

extern "C" int hmx_append_paged_kv8(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                    const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                    const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                    int32_t dtype, void* q_out, int64_t q_out_token_stride,
                                    int64_t q_out_head_stride, const hmx_paged_kv* cache,
                                    const hmx_kv_scales* scales, const void* slots, int32_t slots_int64,
                                    const void* positions, int32_t positions_int64, const void* cos_sin,
                                    int32_t cos_sin_dtype, int64_t cos_sin_stride,
                                    int64_t max_position, int32_t rotary_dim, int32_t interleaved,
                                    int64_t tokens, int32_t H, int32_t HKV, int32_t D,
                                    void* stream) {
  HMX_REQUIRE(scales, HMX_EINVAL, "hmx_append_paged_kv8: no scales");
  return append_paged_kv("hmx_append_paged_kv8", q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v,
                         v_token_stride, v_head_stride, dtype, q_out, q_out_token_stride, q_out_head_stride, cache,
                         scales, slots, slots_int64, positions, positions_int64, cos_sin, cos_sin_dtype,
                         cos_sin_stride, max_position, rotary_dim, interleaved, tokens, H, HKV, D, stream);
}
