// Attention of one new token a sequence over a paged cache:
//   o_n = sum_j softmax_j(scale q_n . k_j) v_j over the sequence's keys j < len_n
// Bound by memory: every key and value is read once, by the workgroup that holds all
// heads of its group (up to 16 columns of a matrix product).
//
// The lengths are known on the device only (a captured step replays with other lengths),
// so the work is cut there: the keys of all sequences, in units of 64, form one list, and
// worker w of W takes units [w per, (w + 1) per).  All workers get the same share whatever
// the lengths are, and a sequence cut over several workers is joined by a second launch
// from fp32 shares.  A worker's four waves take 16 keys in turn; nothing is shared between
// them until a sequence's share ends.  K and V rows go straight into the wave's own ring in
// LDS, whole rows to a load, RING - 1 turns ahead, and are read there as the A operands of
// S^T = K Q^T and (transposed) of O^T = V^T P^T.
// P enters its product as the inputs' type and, beside it, what that rounding leaves: the
// matrix cores wait for memory anyway.  Scores, statistics and O stay in fp32.
//
// Measured: 256 sequences to 8192 keys, 32 / 8 heads of 128 (4.7 GB), 829 us, 5.7 TB/s, where
// a large copy reaches 4.7 - 5.1 (875 us where the rows came through registers); two
// sequences to 131072 keys, 14 / 2 heads of 64, 31 - 35 us with the joining.
#include "attn.hpp"

namespace hmx {
namespace attn {

constexpr int UNIT = 64;     // keys of a unit
constexpr int KT = 16;       // keys of a wave's turn
constexpr int NW = 4;        // waves
constexpr int MIN_UNITS = 4; // of a worker: below that the joining costs more than it gains
// Where a table holds no more keys than this, a worker takes whole sequences: one launch and
// no scan of the lengths (one sequence of 700 keys, 32 / 8 heads: 16.7 us a call where a cut
// and its joining take 19.6).
constexpr int SHORT_KEYS = 1024;

struct DecArgs {
  const char* q;
  char* o;
  int64_t q_ts, q_hs, o_ts, o_hs;   // bytes
  Pages pages;
  int32_t N, HKV, G, hblocks, W;    // hblocks: blocks of 16 heads of a group; W = 0: worker w takes sequence w
  float c;
  float* part;   // [W][2][HKV * hblocks][16][D], then [W][2][HKV * hblocks][16][2]
};

__device__ __forceinline__ int seq_keys(const DecArgs& a, int n) {
  return (int)min((int64_t)max(a.pages.lens[n], 0), (int64_t)a.pages.width * a.pages.page.d);
}

// The list of units, seen by one workgroup: `total` units, and where unit w * per lies, per
// being the workers' share: its sequence and that sequence's first unit.  Every thread adds
// up the sequences of its own run of N / 256.  All threads call it; sh holds 8 int64.
struct Place { int64_t total, per; int seq; int64_t first; };
__device__ __forceinline__ int64_t units_per(const DecArgs& a, int64_t total);
__device__ __forceinline__ Place find_share(const DecArgs& a, int w, int64_t* sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (a.N + 255) >> 8, n0 = min(tid * run, a.N), n1 = min(n0 + run, a.N);
  int64_t mine = 0;
  for (int n = n0; n < n1; ++n) mine += (seq_keys(a, n) + UNIT - 1) / UNIT;
  int64_t x = mine;
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  int64_t before = x - mine;
  for (int i = 0; i < wave; ++i) before += sh[i];
  Place p;
  p.total = sh[0] + sh[1] + sh[2] + sh[3];
  p.per = units_per(a, p.total);
  const int64_t at = w * p.per;
  if (at >= before && at < before + mine) {   // one thread, where there is such a unit
    int n = n0;
    for (int64_t u; (u = (seq_keys(a, n) + UNIT - 1) / UNIT) <= at - before; ++n) before += u;
    sh[4] = n;
    sh[5] = before;
  }
  __syncthreads();
  p.seq = (int)sh[4];
  p.first = sh[5];
  return p;
}

__device__ __forceinline__ int64_t units_per(const DecArgs& a, int64_t total) {
  const int64_t per = (total + a.W - 1) / a.W;
  return per < MIN_UNITS ? MIN_UNITS : per;
}

template <typename T, int D>
__global__ __launch_bounds__(64 * NW) void attn_decode_kernel(DecArgs a) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int NS = D / 32, ND = D / 16, NC = D / 8;
  constexpr int RI = 64 / NC, NL = KT / RI;  // rows of a load, loads of K (and V) of a turn
  constexpr int RING = D == 128 ? 4 : 8;     // turns: 128 KB of LDS for the four waves
  constexpr int KV = KT * D * 2;             // bytes of a turn's K, and of its V behind it
  __shared__ __align__(1024) char smem[NW * RING * 2 * KV];   // the rings, then the shares [16][D] in fp32
  __shared__ float s_ml[NW][16][2];
  __shared__ int64_t s_scan[8];

  const int tid = threadIdx.x, lane = tid & 63, q4 = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hb = blockIdx.x % (a.HKV * a.hblocks), w = blockIdx.x / (a.HKV * a.hblocks);
  const int kvh = hb % a.HKV, g0 = (hb / a.HKV) * 16;
  const int ng = min(16, a.G - g0);

  auto zero_row = [&](int n) {
    for (int i = tid; i < ng * (D / 8); i += 64 * NW)
      *reinterpret_cast<u32x4*>(a.o + (int64_t)n * a.o_ts + (int64_t)(kvh * a.G + g0 + i / (D / 8)) * a.o_hs +
                                16 * (i % (D / 8))) = u32x4{0, 0, 0, 0};
  };
  int seq = __builtin_amdgcn_readfirstlane(w);
  int64_t first = 0, u_beg = 0, u_end;
  if (a.W == 0) {
    u_end = (seq_keys(a, w) + UNIT - 1) / UNIT;
    if (u_end == 0) zero_row(w);
  } else {
    // rows without keys, a worker every W-th sequence
    for (int n = w; n < a.N; n += a.W)
      if (seq_keys(a, n) == 0) zero_row(n);
    const Place pl = find_share(a, w, s_scan);
    u_beg = w * pl.per;
    u_end = min(pl.total, u_beg + pl.per);
    seq = __builtin_amdgcn_readfirstlane(pl.seq);
    first = pl.first;
  }
  if (u_beg >= u_end) return;
  int64_t u = u_beg;

  char* ring = smem + wave * RING * 2 * KV;
  const uint32_t ring_at = lds_addr(ring);
  int ko[NS], vo[ND];                       // the lane's byte offsets into a turn's K and V
#pragma unroll
  for (int s = 0; s < NS; ++s) ko[s] = (l16 * D + swz<D>(l16, 4 * s + q4) * 8) * 2;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int r = 4 * q4 + (l16 >> 2);
    vo[d] = KV + (r * D + swz<D>(r, 2 * d + ((l16 & 3) >> 1)) * 8 + 4 * (l16 & 1)) * 2;
  }
  uint32_t koff[NL], voff[NL];              // and its chunks' offsets from the turn's first row in a page
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = i * RI + lane / NC, c = swz<D>(r, lane % NC);
    koff[i] = (uint32_t)(r * (int)a.pages.k_ts + 16 * c);
    voff[i] = (uint32_t)(r * (int)a.pages.v_ts + 16 * c);
  }
  const char *kbase = a.pages.k + (int64_t)kvh * a.pages.k_hs, *vbase = a.pages.v + (int64_t)kvh * a.pages.v_hs;
  const bool one_page = a.pages.page.d % KT == 0;   // a turn's rows lie in one page

  while (u < u_end) {
    // this worker's share of sequence seq: keys k_beg .. k_end - 1
    int keys = __builtin_amdgcn_readfirstlane(seq_keys(a, seq));
    while (keys == 0) keys = __builtin_amdgcn_readfirstlane(seq_keys(a, ++seq));     // u < total: a sequence with keys follows
    const int64_t units = (keys + UNIT - 1) / UNIT;
    const int k_beg = __builtin_amdgcn_readfirstlane((int)(u - first) * UNIT);
    const int64_t stop = min(u_end, first + units);
    const int k_end = __builtin_amdgcn_readfirstlane(min(keys, (int)(stop - first) * UNIT));
    const int32_t* table = a.pages.table + (int64_t)seq * a.pages.table_stride;

    v8 qf[NS];
    {
      const int hq = kvh * a.G + g0 + min(l16, ng - 1);
      const char* qp = a.q + (int64_t)seq * a.q_ts + (int64_t)hq * a.q_hs + 16 * q4;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const v8*>(qp + 64 * s);
    }
    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEG_INF, l = 0.f;

    // turn x of the wave's: keys k_beg + (x NW + wave) KT ..; live: which of its rows are keys
    const int turns = k_end - k_beg > wave * KT ? (k_end - k_beg - wave * KT + NW * KT - 1) / (NW * KT) : 0;
    uint32_t live[RING];
    auto fetch = [&](int x) __attribute__((always_inline)) {
      const int k0 = k_beg + (x * NW + wave) * KT;
      const uint32_t lds = ring_at + (x % RING) * 2 * KV;
      const int n = k_end - k0;
      uint32_t mask = n >= KT ? (1u << KT) - 1 : (1u << n) - 1;
      if (one_page) {
        // rows behind the last key are the page's own: what they hold is masked
        const int p = __builtin_amdgcn_readfirstlane(fdiv(k0, a.pages.page));
        int id = uniform_load(table, p);
        if ((unsigned)id >= (unsigned)a.pages.num_pages) id = 0, mask = 0;
        const int64_t in = k0 - p * a.pages.page.d;
        const char *kb = uniform_ptr(kbase + id * a.pages.k_ps + in * a.pages.k_ts);
        const char *vb = uniform_ptr(vbase + id * a.pages.v_ps + in * a.pages.v_ts);
#pragma unroll
        for (int i = 0; i < NL; ++i) dma16(lds + i * RI * D * 2, kb, koff[i]);
#pragma unroll
        for (int i = 0; i < NL; ++i) dma16(lds + KV + i * RI * D * 2, vb, voff[i]);
      } else {
        const int mine = min(k0 + l16, k_end - 1);
        mask &= (uint32_t)__ballot((unsigned)table[fdiv(mine, a.pages.page)] < (unsigned)a.pages.num_pages);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int x16 = i * RI + lane / NC, key = min(k0 + x16, k_end - 1), p = fdiv(key, a.pages.page);
          int id = table[p];
          if ((unsigned)id >= (unsigned)a.pages.num_pages) id = 0;
          const int64_t in = key - p * a.pages.page.d;
          const int c = 16 * swz<D>(x16, lane % NC);
          dma16(lds + i * RI * D * 2, kbase + id * a.pages.k_ps + in * a.pages.k_ts + c);
          dma16(lds + KV + i * RI * D * 2, vbase + id * a.pages.v_ps + in * a.pages.v_ts + c);
        }
      }
      return mask;
    };
    // x is a multiple of RING plus the constant i: live[] stays in registers
    auto turn = [&](int x, int i) __attribute__((always_inline)) {
      if (x + RING - 2 < turns) dma_wait<(RING - 2) * 2 * NL>();
      else dma_wait<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the turn before has been read
      char* tile = ring + i * 2 * KV;
      const uint32_t mask = live[i];
      if (x + RING - 1 < turns) live[(i + RING - 1) % RING] = fetch(x + RING - 1);
      if (mask != (1u << KT) - 1) {
        // V rows that are no keys to 0: their probability is 0, their memory anything
#pragma unroll
        for (int z = 0; z < NL; ++z)
          if (!((mask >> (z * RI + lane / NC)) & 1))
            *reinterpret_cast<u32x4*>(tile + KV + (z * 64 + lane) * 16) = u32x4{0, 0, 0, 0};
      }
      f32x4 st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s) st = El<T>::mma16(*reinterpret_cast<const v8*>(tile + ko[s]), qf[s], st);
      if (mask != (1u << KT) - 1) {
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (!((mask >> (4 * q4 + z)) & 1)) st[z] = NEG_INF;
      }
      float mx = fmaxf(fmaxf(st[0], st[1]), fmaxf(st[2], st[3]));
      mx = q4_max(mx);
      if (__any((mx - m) * a.c > 8.f)) {
        const float mn = fmaxf(m, mx);
        const float f = m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
      }
      const float mc = m == NEG_INF ? 0.f : m * a.c;
      v4 pf, pr;                            // P and what its rounding leaves
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float p = __builtin_amdgcn_exp2f(st[z] * a.c - mc);
        l += p;
        pf[z] = (T)p;
        pr[z] = (T)(p - (float)pf[z]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const v4 v = tr4<T>(reinterpret_cast<const T*>(tile + vo[d]));
        acc[d] = El<T>::mma16k16(v, pr, El<T>::mma16k16(v, pf, acc[d]));
      }
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
      if (i < turns) live[i] = fetch(i);
    for (int x = 0; x < turns; x += RING) {
#pragma unroll
      for (int i = 0; i < RING; ++i)
        if (x + i < turns) turn(x + i, i);
    }
    l = q4_sum(l);

    // the waves' shares joined through LDS: O^T rows 16 d + 4 q4 + i, column l16
    __syncthreads();
    float* ob = reinterpret_cast<float*>(smem);       // [wave][16][D]
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<f32x4*>(ob + (wave * 16 + l16) * D + 16 * d + 4 * q4) = acc[d];
    if (q4 == 0) {
      s_ml[wave][l16][0] = m * a.c;
      s_ml[wave][l16][1] = l;
    }
    __syncthreads();
    const bool whole = k_beg == 0 && k_end == keys;
    const int piece = u_beg < first ? 1 : 0;
    const int64_t slot = ((int64_t)w * 2 + piece) * a.HKV * a.hblocks + hb;
    float* pp = a.part + slot * 16 * D;
    float* pm = a.part + (int64_t)a.W * 2 * a.HKV * a.hblocks * 16 * D + slot * 32;
    for (int i = tid; i < ng * (D / 4); i += 64 * NW) {
      const int g = i / (D / 4), d = 4 * (i % (D / 4));
      float mm = NEG_INF, ll = 0.f;
      for (int x = 0; x < NW; ++x) mm = fmaxf(mm, s_ml[x][g][0]);
      const float ref = mm == NEG_INF ? 0.f : mm;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int x = 0; x < NW; ++x) {
        const float f = __builtin_amdgcn_exp2f(s_ml[x][g][0] - ref);
        ll += f * s_ml[x][g][1];
        o += f * *reinterpret_cast<const f32x4*>(ob + (x * 16 + g) * D + d);
      }
      if (whole) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        typename El<T>::v4 y;
#pragma unroll
        for (int z = 0; z < 4; ++z) y[z] = (T)(o[z] * inv);
        *reinterpret_cast<typename El<T>::v4*>(a.o + (int64_t)seq * a.o_ts +
                                               (int64_t)(kvh * a.G + g0 + g) * a.o_hs + 2 * d) = y;
      } else {
        *reinterpret_cast<f32x4*>(pp + g * D + d) = o;
        if (d == 0) {
          pm[2 * g] = mm;
          pm[2 * g + 1] = ll;
        }
      }
    }
    __syncthreads();
    u = stop;
    first += units;
    ++seq;
  }
}

// Sequences cut over several workers: their shares joined.  A workgroup takes one head of
// one sequence; its threads take the shares in turn, D / 4 to a share, and meet in LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_decode_join_kernel(DecArgs a) {
  constexpr int TPS = D / 4, SH = 256 / TPS;
  __shared__ int64_t s_scan[8];
  __shared__ __align__(16) f32x4 s_o[SH][TPS];
  __shared__ float s_ml[SH][2];
  const int H = a.HKV * a.G, head = blockIdx.x % H, n = blockIdx.x / H;
  const int kvh = head / a.G, g = head - kvh * a.G, hb = (g >> 4) * a.HKV + kvh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int keys = seq_keys(a, n);
  if (keys <= UNIT) return;                 // one unit is never cut
  int64_t before = 0, total = 0;            // units before sequence n, and of all
  for (int x = tid; x < a.N; x += 256) {
    const int64_t u = (seq_keys(a, x) + UNIT - 1) / UNIT;
    total += u;
    if (x < n) before += u;
  }
  for (int d = 32; d >= 1; d >>= 1) {
    before += __shfl_xor(before, d, 64);
    total += __shfl_xor(total, d, 64);
  }
  if (lane == 0) {
    s_scan[tid >> 6] = before;
    s_scan[4 + (tid >> 6)] = total;
  }
  __syncthreads();
  before = s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3];
  total = s_scan[4] + s_scan[5] + s_scan[6] + s_scan[7];
  const int64_t per = units_per(a, total), last = before + (keys + UNIT - 1) / UNIT - 1;
  const int w0 = (int)(before / per), w1 = (int)(last / per);
  if (w0 == w1) return;
  const int64_t hbs = (int64_t)a.HKV * a.hblocks, stats = (int64_t)a.W * 2 * hbs * 16 * D;
  const int d = tid % TPS, sh = tid / TPS;
  float m = NEG_INF, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int w = w0 + sh; w <= w1; w += SH) {
    const int64_t slot = ((int64_t)w * 2 + (w * per < before ? 1 : 0)) * hbs + hb;
    const float* ml = a.part + stats + slot * 32 + 2 * (g & 15);
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + (slot * 16 + (g & 15)) * D + 4 * d);
    const float mn = fmaxf(m, ml[0]), ref = mn == NEG_INF ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(ml[0] - ref);
    l = l * f + ml[1] * e;
    o = o * f + x * e;
    m = mn;
  }
  s_o[sh][d] = o;
  if (d == 0) {
    s_ml[sh][0] = m;
    s_ml[sh][1] = l;
  }
  __syncthreads();
  if (sh == 0) {
    for (int i = 1; i < SH; ++i) {
      const float mi = s_ml[i][0], mn = fmaxf(m, mi), ref = mn == NEG_INF ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(mi - ref);
      l = l * f + s_ml[i][1] * e;
      o = o * f + s_o[i][d] * e;
      m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typename El<T>::v4 y;
#pragma unroll
    for (int z = 0; z < 4; ++z) y[z] = (T)(o[z] * inv);
    *reinterpret_cast<typename El<T>::v4*>(a.o + (int64_t)n * a.o_ts + (int64_t)head * a.o_hs + 8 * d) = y;
  }
}

// Workers: as many as there are compute units (a workgroup fills one's LDS), and no more than
// the keys a table can hold give MIN_UNITS to.
static int64_t workers(int64_t N, int64_t HKV, int64_t hblocks, int64_t max_keys) {
  if (max_keys <= SHORT_KEYS) return 0;
  const int64_t most = N * ((max_keys + UNIT - 1) / UNIT);
  int64_t w = cu_count() / (HKV * hblocks);
  const int64_t need = (most + MIN_UNITS - 1) / MIN_UNITS;
  if (w > need) w = need;
  return w < 1 ? 1 : w;
}

template <typename T, int D>
static void launch(const DecArgs& a, bool join, hipStream_t s) {
  const unsigned hbs = (unsigned)(a.HKV * a.hblocks);
  hipLaunchKernelGGL((attn_decode_kernel<T, D>), dim3(hbs * (unsigned)(a.W ? a.W : a.N)), dim3(64 * NW), 0, s, a);
  if (join)
    hipLaunchKernelGGL((attn_decode_join_kernel<T, D>), dim3((unsigned)(a.HKV * a.G * a.N)), dim3(256), 0, s, a);
}

}  // namespace attn
}  // namespace hmx

using namespace hmx;

extern "C" size_t hmx_paged_attention_decode_workspace_bytes(int32_t N, int32_t H, int32_t HKV,
                                                             int32_t D, int64_t max_keys) {
  if (N <= 0 || HKV <= 0 || H <= 0 || H % HKV != 0 || max_keys <= 0) return 0;
  const int64_t hb = (H / HKV + 15) / 16, w = attn::workers(N, HKV, hb, max_keys);
  if (w <= 1) return 0;
  return (size_t)w * 2 * HKV * hb * 16 * (D + 2) * sizeof(float);
}

extern "C" int hmx_paged_attention_decode(const void* q, int64_t q_token_stride,
                                          int64_t q_head_stride, int32_t dtype, void* o,
                                          int64_t o_token_stride, int64_t o_head_stride,
                                          const hmx_paged_kv* cache, int32_t N, int32_t H,
                                          int32_t HKV, int32_t D, float scale, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  HMX_REQUIRE(D == 64 || D == 128, HMX_EUNSUPPORTED,
              "hmx_paged_attention_decode: head size %d not in {64, 128}", D);
  HMX_REQUIRE(dtype == HMX_BF16 || dtype == HMX_F16, HMX_EUNSUPPORTED,
              "hmx_paged_attention_decode: dtype code %d (bf16 or fp16)", dtype);
  HMX_REQUIRE(N >= 0 && HKV > 0 && H > 0 && H % HKV == 0, HMX_EINVAL,
              "hmx_paged_attention_decode: N=%d H=%d HKV=%d", N, H, HKV);
  HMX_REQUIRE(scale > 0.f && scale < __builtin_inff(), HMX_EINVAL,
              "hmx_paged_attention_decode: scale %g must be positive", (double)scale);
  HMX_REQUIRE(cache && cache->num_pages >= 0 && cache->page_size > 0 && cache->table_width >= 0, HMX_EINVAL,
              "hmx_paged_attention_decode: cache");
  if (N == 0) return HMX_OK;
  HMX_REQUIRE(q && o && cache->seq_lens && attn::has_pages(*cache), HMX_EINVAL,
              "hmx_paged_attention_decode: null pointer");
  const int64_t max_keys = (int64_t)cache->table_width * cache->page_size;
  HMX_REQUIRE(max_keys < (1ll << 31) - 256, HMX_EUNSUPPORTED,
              "hmx_paged_attention_decode: a table row holds %lld keys", (long long)max_keys);
  const int64_t st = q_token_stride | q_head_stride | o_token_stride | o_head_stride |
                     cache->k_page_stride | cache->k_token_stride | cache->k_head_stride |
                     cache->v_page_stride | cache->v_token_stride | cache->v_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)o | (uintptr_t)cache->k | (uintptr_t)cache->v;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0, HMX_EINVAL,
              "hmx_paged_attention_decode: strides must be multiples of 8 elements and pointers 16-byte aligned");
  HMX_REQUIRE(attn::near_rows(cache->k_token_stride) && attn::near_rows(cache->v_token_stride), HMX_EUNSUPPORTED,
              "hmx_paged_attention_decode: token strides of the cache past 2^25 elements");
  attn::DecArgs a{};
  a.q = (const char*)q; a.o = (char*)o;
  a.q_ts = 2 * q_token_stride; a.q_hs = 2 * q_head_stride;
  a.o_ts = 2 * o_token_stride; a.o_hs = 2 * o_head_stride;
  a.pages = attn::make_pages(*cache);
  a.N = N; a.HKV = HKV; a.G = H / HKV; a.hblocks = (a.G + 15) / 16;
  a.W = (int32_t)attn::workers(N, HKV, a.hblocks, max_keys);
  a.c = scale * attn::LOG2E;
  a.part = static_cast<float*>(workspace);
  HMX_REQUIRE((int64_t)N * H < (1ll << 31), HMX_EUNSUPPORTED,
              "hmx_paged_attention_decode: %d sequences of %d heads", N, H);
  const bool join = a.W > 1;
  HMX_REQUIRE(!join || (workspace && (uintptr_t)workspace % 16 == 0 &&
                        workspace_bytes >= hmx_paged_attention_decode_workspace_bytes(N, H, HKV, D, max_keys)),
              HMX_EINVAL, "hmx_paged_attention_decode: workspace of %zu bytes is too small", workspace_bytes);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == HMX_BF16) {
    if (D == 64) attn::launch<bf16, 64>(a, join, s);
    else attn::launch<bf16, 128>(a, join, s);
  } else {
    if (D == 64) attn::launch<f16, 64>(a, join, s);
    else attn::launch<f16, 128>(a, join, s);
  }
  return check_launch("hmx_paged_attention_decode");
}
