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
// 842 - 902 us, 0.91 - 0.98, over a cache of 8 bits 949 - 987, 0.83 - 0.87; draft tokens of eight
// sequences to 16384 keys 63 - 75 us and the joining 6 (76 us where every sequence's keys were cut
// into as many splits).
#include "attn_tile.hpp"

namespace hmx {
namespace attn {

template <typename T, int D, bool PAGED, bool Q8 = false>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_fwd_kernel(FwdArgs a) {
  constexpr bool PREFIX = false;
  __shared__ __align__(1024) char smem[tile_bytes<D, Q8>()];
  __shared__ int s_bad, s_skip[4];
  const unsigned block = blockIdx.x, blocks = gridDim.x;
#include "attn_tile_body.hpp"
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

template <typename T, bool PAGED, bool Q8 = false>
static void launch_fwd(FwdArgs a, int D, hipStream_t s) {
  a.places = (int32_t)(cu_count() / a.HKV);
  const int64_t blocks = fwd_blocks(a);
  const dim3 grid((unsigned)(blocks * a.HKV));
  if (D == 64) hipLaunchKernelGGL((attn_fwd_kernel<T, 64, PAGED, Q8>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((attn_fwd_kernel<T, 128, PAGED, Q8>), grid, dim3(256), 0, s, a);
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

extern "C" size_t hmx_paged_causal_attention8_workspace_bytes(int32_t N, int64_t T, int32_t H,
                                                              int32_t HKV, int32_t D,
                                                              int64_t max_keys) {
  if (N <= 0 || T <= 0 || HKV <= 0 || H <= 0 || H % HKV != 0 || max_keys < 0) return 0;
  return attn::few_rows(N, T, H / HKV) ? attn::few_rows_workspace_bytes(N, T, H, HKV, D, max_keys)
                                       : hmx_paged_causal_attention_workspace_bytes(N, T, H, HKV, D, max_keys);
}

static int paged_causal_attention(const void* q, int64_t q_token_stride,
                                  int64_t q_head_stride, int32_t dtype, void* o,
                                  int64_t o_token_stride, int64_t o_head_stride,
                                  const hmx_paged_kv* cache, const hmx_kv_scales* scales,
                                  const int32_t* cu_seqlens,
                                  int32_t N, int64_t T, int32_t H, int32_t HKV, int32_t D,
                                  float scale, int32_t fill_gaps, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  ATTN_COMMON_CHECKS("hmx_paged_causal_attention")
  HMX_REQUIRE(cache && cache->num_pages >= 0 && cache->page_size > 0 && cache->table_width >= 0, HMX_EINVAL,
              "hmx_paged_causal_attention: cache");
  if (T == 0) return HMX_OK;
  HMX_REQUIRE(q && o && cu_seqlens && (N == 0 || (cache->seq_lens && attn::has_pages(*cache) &&
                                                     attn::has_scales(*cache, scales))),
              HMX_EINVAL, "hmx_paged_causal_attention: null pointer");
  const int64_t max_keys = (int64_t)cache->table_width * cache->page_size;
  HMX_REQUIRE(max_keys < (1ll << 31) - 256, HMX_EUNSUPPORTED,
              "hmx_paged_causal_attention: a table row holds %lld keys", (long long)max_keys);
  const int64_t st = q_token_stride | q_head_stride | o_token_stride | o_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)o;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0 && attn::aligned_pages(*cache, scales != nullptr), HMX_EINVAL,
              "hmx_paged_causal_attention: strides must be multiples of 8 elements (a cache's of 16 bytes) and "
              "pointers 16-byte aligned");
  HMX_REQUIRE(attn::near_rows(cache->k_token_stride) && attn::near_rows(cache->v_token_stride), HMX_EUNSUPPORTED,
              "hmx_paged_causal_attention: token strides of the cache past 2^25 elements");
  const size_t need = scales ? hmx_paged_causal_attention8_workspace_bytes(N, T, H, HKV, D, max_keys)
                             : hmx_paged_causal_attention_workspace_bytes(N, T, H, HKV, D, max_keys);
  HMX_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need), HMX_EINVAL,
              "hmx_paged_causal_attention: workspace of %zu bytes is too small", workspace_bytes);
  if (scales && attn::few_rows(N, T, H / HKV)) {
    HMX_REQUIRE(T * H < (1ll << 31) && (int64_t)N * H < (1ll << 30), HMX_EUNSUPPORTED,
                "hmx_paged_causal_attention8: %lld tokens of %d sequences", (long long)T, N);
    attn::launch_few_rows(attn::FewRows{q, o, q_token_stride, q_head_stride, o_token_stride, o_head_stride, dtype,
                                        attn::make_pages(*cache, scales), cu_seqlens, N, (int32_t)T, H, HKV, D, max_keys,
                                        scale, fill_gaps, static_cast<float*>(workspace)},
                          (hipStream_t)stream);
    return check_launch("hmx_paged_causal_attention8");
  }
  attn::FwdArgs a{};
  a.q = (const char*)q; a.o = (char*)o;
  a.q_ts = 2 * q_token_stride; a.q_hs = 2 * q_head_stride;
  a.o_ts = 2 * o_token_stride; a.o_hs = 2 * o_head_stride;
  a.seqs = attn::Seqs{cu_seqlens, N, (int32_t)T, H / HKV};
  a.G = attn::fast_div(H / HKV);
  a.pages = attn::make_pages(*cache, scales);
  const int64_t slots = attn::tile_slots<attn::BM>(cu_seqlens, N, T, H / HKV);
  HMX_REQUIRE(slots * HKV < (1ll << 31), HMX_EUNSUPPORTED, "hmx_paged_causal_attention: %lld tiles",
              (long long)slots);
  a.H = H; a.HKV = HKV; a.slots = (int32_t)slots; a.fill = fill_gaps;
  a.split = N == 0 ? attn::NO_SPLITS : paged_splits(N, T, H, HKV, max_keys);
  a.nsplit = a.split.most;
  a.part = static_cast<float*>(workspace);
  a.c = scale * attn::LOG2E;
  hipStream_t st_ = (hipStream_t)stream;
  if (dtype == HMX_BF16) {
    if (scales) attn::launch_fwd<bf16, true, true>(a, D, st_);
    else attn::launch_fwd<bf16, true>(a, D, st_);
  } else {
    if (scales) attn::launch_fwd<f16, true, true>(a, D, st_);
    else attn::launch_fwd<f16, true>(a, D, st_);
  }
  return check_launch("hmx_paged_causal_attention");
}

extern "C" int hmx_paged_causal_attention(const void* q, int64_t q_token_stride,
                                          int64_t q_head_stride, int32_t dtype, void* o,
                                          int64_t o_token_stride, int64_t o_head_stride,
                                          const hmx_paged_kv* cache, const int32_t* cu_seqlens,
                                          int32_t N, int64_t T, int32_t H, int32_t HKV, int32_t D,
                                          float scale, int32_t fill_gaps, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  return paged_causal_attention(q, q_token_stride, q_head_stride, dtype, o, o_token_stride, o_head_stride, cache,
                                nullptr, cu_seqlens, N, T, H, HKV, D, scale, fill_gaps, workspace, workspace_bytes,
                                stream);
}

extern "C" int hmx_paged_causal_attention8(const void* q, int64_t q_token_stride,
                                           int64_t q_head_stride, int32_t dtype, void* o,
                                           int64_t o_token_stride, int64_t o_head_stride,
                                           const hmx_paged_kv* cache, const hmx_kv_scales* scales,
                                           const int32_t* cu_seqlens,
                                           int32_t N, int64_t T, int32_t H, int32_t HKV, int32_t D,
                                           float scale, int32_t fill_gaps, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  HMX_REQUIRE(scales, HMX_EINVAL, "hmx_paged_causal_attention8: no scales");
  return paged_causal_attention(q, q_token_stride, q_head_stride, dtype, o, o_token_stride, o_head_stride, cache,
                                scales, cu_seqlens, N, T, H, HKV, D, scale, fill_gaps, workspace, workspace_bytes,
                                stream);
}
