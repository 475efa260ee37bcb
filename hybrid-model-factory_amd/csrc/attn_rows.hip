// Attention of few rows over long contexts in pages:
// - one new token a sequence, or a few (draft tokens), over a cache of 8 bits;
// - one new token a sequence behind prefixes that groups of sequences share, in 8 bits or 16.
//   o_r = sum_j softmax_j(scale q_r . k_j) v_j  over the keys that row r attends
// Bound by memory: every key and value is read once for 16 rows, the columns of a matrix
// product; a row is (token, head of the group) of one key/value head.
//
// The lengths are known on the device only, so the work is cut there.  An entry is a sequence,
// or a prefix with all tokens behind it: its rows, in blocks of 16, times its keys, in units of
// 64.  The units of all blocks of all entries form one list, with SETUP more before a block's
// keys for what its beginning costs, and worker w of W takes units [w per, (w + 1) per): all get
// the same share whatever the lengths are.  A block cut over
// several workers, and a row that has both a prefix and keys of its own, are joined by a second
// launch from fp32 shares.
//
// A worker's four waves take KT keys in turn; nothing is shared between them until a block's
// share ends.  K and V rows go straight into the wave's own ring in LDS, RING - 1 turns ahead,
// and are read there as the A operands of S^T = K Q^T and (transposed) of O^T = V^T P^T.  Where
// they lie is formed for 64 times 16 keys at once, a lane each.
// A cache of 8 bits is widened where its fragments are read (every e4m3 value is a bf16 and an
// fp16 value); a key's scale multiplies its scores, and its probabilities before their product
// with V, both in fp32, so neither type's range matters.  V's fragments come from the
// transposing read of bytes: eight keys of one column, four of the first sixteen keys of a turn
// and four of the second, the order in which the two tiles of scores hold them.
// P enters its product rounded and, beside it, what that rounding leaves: the matrix cores wait
// for memory anyway.  Scores, statistics and O stay in fp32.
//
// Measured, in 8 bits, 32 / 8 heads of 128: 256 sequences to 8192 keys 397 us alone (6.0 TB/s, a
// part of the cache kept from the call before) and 472 a call with other caches read in between;
// eight of up to four tokens to 16384 keys 38 - 44; one of 700 keys 12.7; two to 131072 keys, 14 / 2
// heads of 64, 20; the joining launch 6 - 11.  Behind prefixes: eight to 129 keys behind 4096 13,
// 256 to 1031 keys in 16 bits behind two to 16384 178, where one read of all and the products
// alone would take 139.
#include "attn_rows_plan.hpp"
#include "attn_tile.hpp"

namespace hmx {
namespace attn {
namespace rows {

constexpr int UNIT = 64;     // keys of a unit
constexpr int NW = 4;        // waves
// Workgroups of a compute unit: while one finds its next block, joins its waves or waits for
// its first rows the other streams (256 sequences to 1031 keys, 32 / 8 heads of 128: 146 -> 106 us;
// to 8192 keys 527 -> 497; one workgroup of eight waves 138 and 499).
constexpr int OCC = 2;
// What beginning a block costs, in units: it stands in the list as so many before its keys, so
// workers with many short blocks get fewer keys (the same batch 89.5 -> 83.7 us with 4, 81.7 with
// 8; eight sequences to 129 keys behind one prefix of 4096 35 -> 21 either way).
constexpr int SETUP = 4;
constexpr int MIN_UNITS = 4; // of a worker: below that the joining costs more than it gains
// Where a table holds no more keys than this, a worker takes one sequence, or of several tokens
// one block: one launch, and no scan of the lengths (64 sequences to 1024 keys, 32 / 8 heads of
// 128, 4 tokens each 28 us, cut evenly and joined 36; one of 190 tokens among 63 of one 40, 43,
// by whole sequences 585).
constexpr int SHORT_KEYS = 1024;

struct Args {
  const char* q;
  char* o;
  int64_t q_ts, q_hs, o_ts, o_hs;   // bytes
  Pages pages;                      // of the sequences
  const int32_t* cu;                // their tokens; NULL: sequence n has token n alone
  const int32_t *p_table, *p_lens, *p_cu;   // M prefixes (p_cu NULL: one for all tokens)
  int64_t p_stride;
  int32_t p_width, M, N, T, HKV, W; // W = 0: worker w takes sequence w, or with cu the w-th block
  int32_t blocks;                   // workgroups of a key/value head
  FastDiv G;
  float c;                          // scale log2(e)
  int32_t fill;                     // rows of no sequence become 0
  float* part;   // [slots][HKV][16][D], then [slots][HKV][16][2]
  int64_t slots; // two a worker; where all shares are kept, a block's own behind them
};

struct Entry { int bos, tokens, keys; };
__device__ __forceinline__ int bound(const int32_t* cu, int i, int T) { return min(max(cu[i], 0), T); }
__device__ __forceinline__ Entry entry_of(const Args& a, int e) {
  Entry x;
  const bool prefix = e < a.M;
  const int n = prefix ? e : e - a.M;
  const int32_t* cu = prefix ? a.p_cu : a.cu;
  if (cu) {
    x.bos = bound(cu, n, a.T);
    x.tokens = max(bound(cu, n + 1, a.T) - x.bos, 0);
  } else {
    x.bos = prefix ? 0 : n;
    x.tokens = prefix ? a.T : 1;
  }
  x.keys = (int)min((int64_t)max((prefix ? a.p_lens : a.pages.lens)[n], 0),
                    (int64_t)(prefix ? a.p_width : a.pages.width) * a.pages.page.d);
  return x;
}
__device__ __forceinline__ int units_of(const Entry& x) { return (x.keys + UNIT - 1) / UNIT; }
__device__ __forceinline__ int blocks_of(const Args& a, const Entry& x) { return (int)(((int64_t)x.tokens * a.G.d + 15) >> 4); }
__device__ __forceinline__ int64_t work_of(const Args& a, const Entry& x) {
  return x.keys > 0 ? (int64_t)(units_of(x) + SETUP) * blocks_of(a, x) : 0;
}
__device__ __forceinline__ int64_t units_per(const Args& a, int64_t total) {
  const int64_t per = (total + a.W - 1) / a.W;
  return per < MIN_UNITS ? MIN_UNITS : per;
}
// Where all shares are kept, that of a block which is not cut: behind the workers', the
// sequences' (one token each) and then the prefixes', of which entry e's begin at slot
// bos G / 16 + e, so none meet.
__device__ __forceinline__ int64_t own_slot(const Args& a, int e, const Entry& x, int b) {
  const int per = (a.G.d + 15) >> 4;
  return 2ll * a.W + (e >= a.M ? (int64_t)(e - a.M) * per + b
                               : (int64_t)a.N * per + (((int64_t)x.bos * a.G.d) >> 4) + e + b);
}

// A list of the entries' work, seen by one workgroup: the total, and where unit at(total) lies:
// its entry and that entry's first unit (none past the total: nothing to rely on).  Every thread
// adds up the entries of its own run.  All threads call it; sh holds 8 int64.
struct Place { int64_t total, at; int entry; int64_t first; };
template <typename Work, typename At>
__device__ __forceinline__ Place find_place(int E, Work work, At at_of, int64_t* sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (E + 255) >> 8, n0 = min(tid * run, E), n1 = min(n0 + run, E);
  int64_t mine = 0;
  for (int n = n0; n < n1; ++n) mine += work(n);
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
  p.at = at_of(p.total);
  if (p.at >= before && p.at < before + mine) {   // one thread, where there is such a unit
    int n = n0;
    for (int64_t u; (u = work(n)) <= p.at - before; ++n) before += u;
    sh[4] = n;
    sh[5] = before;
  }
  __syncthreads();
  p.entry = (int)sh[4];
  p.first = sh[5];
  return p;
}

template <int D> __device__ __forceinline__ int swz8k(int r, int c) {   // rows read eight at a time at one chunk
  return D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
}
template <int D> __device__ __forceinline__ int swz8v(int r, int c) {   // rows 4 i .. 4 i + 3 and 16 on at one chunk
  return D == 128 ? c ^ ((r & 3) | (r >> 2 & 4)) : c ^ ((r >> 1 & 1) | (r >> 3 & 2));
}
// The transposing LDS read of bytes: the 16 lanes of a group address eight rows of 16 bytes,
// two lanes to a row, and lane i receives column i of the eight.
__device__ __forceinline__ u32x2 tr8(const char* p) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(p)));
}
// The ring of a wave: turns of KT keys, K's bytes, V's behind them, then the scales.
template <int D, bool Q8, int RING> struct Shared {
  static constexpr int KT = Q8 ? 32 : 16;
  static constexpr int KV = KT * D * (Q8 ? 1 : 2), TURN = 2 * KV + (Q8 ? 256 : 0);
  static constexpr int BYTES = NW * RING * TURN;     // the rings, then the shares [16][D] in fp32
  static_assert(NW == 4 && RING * TURN >= 16 * D * 4, "find_place, and the shares in LDS");
  float ml[NW][16][2];
  int64_t scan[8];
  int bad;                                  // the last share of whose keys some were spoiled
};

// Q8: a cache of 8 bits.  SHARES: every block leaves its share.
template <typename T, int D, bool Q8, bool SHARES, int RING>
__device__ __forceinline__ void attn_rows(const Args& a, char* smem, Shared<D, Q8, RING>& shared, int blk) {
  typedef typename El<T>::v8 v8;
  typedef typename El<T>::v4 v4;
  constexpr int KT = Shared<D, Q8, RING>::KT;  // keys of a wave's turn
  constexpr int ES = Q8 ? 1 : 2;             // bytes of an element of the cache
  constexpr int ROW = D * ES;                // bytes of a row
  constexpr int NH = KT / 16;                // halves of a turn: sixteen keys, one page where pages are of sixteens
  constexpr int NS = D / 32, ND = D / 16, NC = ROW / 16;
  constexpr int RI = 64 / NC, NL = KT / RI;  // rows of a load, loads of K (and V) of a turn
  constexpr int KV = Shared<D, Q8, RING>::KV, TURN = Shared<D, Q8, RING>::TURN;
  constexpr uint32_t ALL = Q8 ? ~0u : 0xffffu;
  auto& s_ml = shared.ml;
  auto& s_scan = shared.scan;
  int& s_bad = shared.bad;

  const int tid = threadIdx.x, lane = tid & 63, q4 = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.G.d;
  // Workgroups go to the eight XCDs in turn.  Rows of 64 bytes are half a cache line, the other
  // half another head's: there the heads of a worker go to one XCD, whose L2 then reads the
  // line once (two sequences to 131072 keys, 14 / 2 heads of 64: 38.5 -> 29.7 us); rows of whole
  // lines are better spread (256 sequences to 8192 keys: 483 us, by worker 500).
  constexpr bool BY_WORKER = ROW < 128;
  constexpr bool ONCE = !SHARES && ROW >= 128;   // (a prefix is read by several blocks)
  const int eights = BY_WORKER ? a.blocks & ~7 : 0;
  const bool in8 = blk < eights * a.HKV;
  const int rem = in8 ? blk % (8 * a.HKV) : blk - eights * a.HKV;
  const int kvh = in8 ? rem >> 3 : rem % a.HKV;
  const int w = in8 ? blk / (8 * a.HKV) * 8 + (rem & 7) : eights + rem / a.HKV;

  auto zero_rows = [&](int t0, int t1) {     // of this key/value head's group
    for (int64_t i = tid; i < (int64_t)(t1 - t0) * G * (D / 8); i += 64 * NW) {
      const int r = (int)(i / (D / 8)), tok = fdiv(r, a.G);
      *reinterpret_cast<u32x4*>(a.o + (int64_t)(t0 + tok) * a.o_ts + (int64_t)(kvh * G + r - tok * G) * a.o_hs +
                                16 * (i % (D / 8))) = u32x4{0, 0, 0, 0};
    }
  };
  int e = __builtin_amdgcn_readfirstlane(w);
  int64_t first = 0, u_beg = 0, u_end;
  if (tid == 0) s_bad = 0;
  if (!SHARES && a.cu && a.fill) {           // rows of no sequence, a workgroup every so many tokens
    const int beg = bound(a.cu, 0, a.T), end = bound(a.cu, a.N, a.T);
    for (int t = w; t < beg; t += a.blocks) zero_rows(t, t + 1);
    for (int t = end + w; t < a.T; t += a.blocks) zero_rows(t, t + 1);
  }
  if (!SHARES && a.W == 0 && !a.cu) {
    const Entry x = entry_of(a, w);
    u_end = work_of(a, x);
    if (x.keys == 0) zero_rows(x.bos, x.bos + x.tokens);
    __syncthreads();                        // s_bad is clear
  } else if (!SHARES && a.W == 0) {         // of all sequences' blocks the w-th
    const Place pl = find_place(a.N, [&](int n) { return (int64_t)blocks_of(a, entry_of(a, n)); },
                                [&](int64_t) { return (int64_t)w; }, s_scan);
    if (pl.at >= pl.total) return;
    e = __builtin_amdgcn_readfirstlane(pl.entry);
    const Entry x = entry_of(a, e);
    const int b = (int)(pl.at - pl.first);
    if (x.keys == 0 && b == 0) zero_rows(x.bos, x.bos + x.tokens);
    u_beg = (int64_t)b * (units_of(x) + SETUP);
    u_end = x.keys == 0 ? u_beg : u_beg + units_of(x) + SETUP;
  } else {
    // rows without keys, a worker every W-th sequence
    if (!SHARES)
      for (int n = w; n < a.N; n += a.W) {
        const Entry x = entry_of(a, n);
        if (x.keys == 0) zero_rows(x.bos, x.bos + x.tokens);
      }
    int64_t per = 0;
    const Place pl = find_place(a.M + a.N, [&](int n) { return work_of(a, entry_of(a, n)); },
                                [&](int64_t total) { return w * (per = units_per(a, total)); }, s_scan);
    u_beg = pl.at;
    u_end = min(pl.total, u_beg + per);
    e = __builtin_amdgcn_readfirstlane(pl.entry);
    first = pl.first;
  }
  if (u_beg >= u_end) return;
  int64_t u = u_beg;

  char* ring = smem + wave * RING * TURN;
  const uint32_t ring_at = lds_addr(ring);
  int ko[NS], vo[ND];                       // the lane's byte offsets into a turn's K and V
  if constexpr (Q8) {                       // a lane reads the sixteen elements of two steps at once
#pragma unroll
    for (int p = 0; p < NS / 2; ++p) ko[p] = l16 * D + swz8k<D>(l16, 4 * p + q4) * 16;   // (row 16 + l16: the same chunk)
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int i = l16 >> 1, r = 4 * q4 + (i & 3) + (i & 4) * 4;
      vo[d] = KV + r * D + swz8v<D>(r, d) * 16 + 8 * (l16 & 1);
    }
  } else {
#pragma unroll
    for (int s = 0; s < NS; ++s) ko[s] = (l16 * D + swz<D>(l16, 4 * s + q4) * 8) * 2;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int r = 4 * q4 + (l16 >> 2);
      vo[d] = KV + (r * D + swz<D>(r, 2 * d + ((l16 & 3) >> 1)) * 8 + 4 * (l16 & 1)) * 2;
    }
  }
  auto kchunk = [](int r, int c) __attribute__((always_inline)) { return 16 * (Q8 ? swz8k<D>(r, c) : swz<D>(r, c)); };
  auto vchunk = [](int r, int c) __attribute__((always_inline)) { return 16 * (Q8 ? swz8v<D>(r, c) : swz<D>(r, c)); };
  const char *kbase = a.pages.k + (int64_t)kvh * a.pages.k_hs, *vbase = a.pages.v + (int64_t)kvh * a.pages.v_hs;
  // lanes 0 .. 31 bring the scales of the keys, 32 .. 63 of the values
  const uint8_t* sbase = lane < 32 ? a.pages.k_sc + kvh * a.pages.k_sc_hs : a.pages.v_sc + kvh * a.pages.v_sc_hs;
  const int64_t sps = lane < 32 ? a.pages.k_sc_ps : a.pages.v_sc_ps;
  const bool whole_pages = a.pages.page.d % 16 == 0;   // sixteen rows of a turn lie in one page

  for (int share = 1; u < u_end; ++share) {
    // this worker's share of entry e's block b: keys k_beg .. k_end - 1
    Entry x = entry_of(a, e);
    while (work_of(a, x) == 0) x = entry_of(a, ++e);     // u < total: an entry with work follows
    x.bos = __builtin_amdgcn_readfirstlane(x.bos);
    x.tokens = __builtin_amdgcn_readfirstlane(x.tokens);
    const int keys = __builtin_amdgcn_readfirstlane(x.keys), units = units_of(x);
    const int len = units + SETUP;          // of the block in the list
    const int b = __builtin_amdgcn_readfirstlane((int)((u - first) / len));
    const int64_t bfirst = first + (int64_t)b * len;
    const int64_t stop = min(u_end, bfirst + len);
    const int k_beg = __builtin_amdgcn_readfirstlane(max((int)(u - bfirst) - SETUP, 0) * UNIT);
    const int k_end = __builtin_amdgcn_readfirstlane(min(keys, ((int)(stop - bfirst) - SETUP) * UNIT));
    u = stop;
    const int e_now = e;
    if (stop == bfirst + len && b + 1 == blocks_of(a, x)) {
      first += (int64_t)len * (b + 1);
      ++e;
    }
    if (k_beg >= k_end) continue;           // none of its keys
    const bool prefix = e_now < a.M;
    const int32_t* table = prefix ? a.p_table + (int64_t)e_now * a.p_stride
                                  : a.pages.table + (int64_t)(e_now - a.M) * a.pages.table_stride;
    const int nrows = min(16, x.tokens * G - 16 * b);
    // the lane's row; token i of n attends keys 0 .. keys - n + i, behind a prefix all
    const int row = 16 * b + min(l16, nrows - 1), tok = fdiv(row, a.G);
    const int klast = prefix ? keys - 1 : keys - x.tokens + tok;
    const int kfirst = prefix ? keys - 1 : keys - x.tokens + __builtin_amdgcn_readfirstlane(fdiv(16 * b, a.G));   // the least of the block

    v8 qf[NS];
    {
      const char* qp = a.q + (int64_t)(x.bos + tok) * a.q_ts + (int64_t)(kvh * G + row - tok * G) * a.q_hs;
#pragma unroll
      for (int s = 0; s < NS; ++s)          // of 8 bits step 2 p takes the first eight of the lane's sixteen, 2 p + 1 the others
        qf[s] = *reinterpret_cast<const v8*>(Q8 ? qp + 32 * q4 + 128 * (s >> 1) + 16 * (s & 1) : qp + 16 * q4 + 64 * s);
    }
    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEG_INF, l = 0.f;
    bool bad = false;

    // turn x of the wave's: keys k_beg + (x NW + wave) KT ..; live: which of its rows are keys
    const int turns = k_end - k_beg > wave * KT ? (k_end - k_beg - wave * KT + NW * KT - 1) / (NW * KT) : 0;
    uint32_t live[RING];
    // The places of 64 halves on: lane i holds half i's first row of K and of V, its page and the
    // row's place there; good: the halves whose pages lie in the cache.  The pages' numbers are
    // asked for 64 halves ahead, and arrive with rows that are waited for anyway.
    constexpr int TURNS = 64 / NH;
    const char *kat = nullptr, *vat = nullptr;
    int at_id = 0, at_in = 0, ahead = 0;
    uint64_t good = 0;
    auto row_at = [&](int x) __attribute__((always_inline)) {   // of the lane's half; the last key's where it lies behind it
      return half_row<NW, KT>(k_beg, k_end, x + lane / NH, wave, lane % NH);
    };
    auto places = [&](int x) __attribute__((always_inline)) {
      const int r = row_at(x), p = fdiv(r, a.pages.page);
      const bool in_cache = (unsigned)ahead < (unsigned)a.pages.num_pages;
      at_id = in_cache ? ahead : 0;
      at_in = r - p * a.pages.page.d;
      good = __ballot(in_cache);
      kat = kbase + at_id * a.pages.k_ps + at_in * a.pages.k_ts;
      vat = vbase + at_id * a.pages.v_ps + at_in * a.pages.v_ts;
      ahead = table[fdiv(row_at(x + TURNS), a.pages.page)];
    };
    auto lane_ptr = [&](const char* p, int i) __attribute__((always_inline)) {
      const uint64_t x = (uint64_t)p;
      return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, i) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32);
    };
    if (whole_pages) ahead = table[fdiv(row_at(0), a.pages.page)];
    auto fetch = [&](int x) __attribute__((always_inline)) {
      const int k0 = k_beg + (x * NW + wave) * KT;
      const uint32_t lds = ring_at + (x % RING) * TURN;
      const int n = k_end - k0;
      uint32_t mask = n >= KT ? ALL : (1u << n) - 1;
      if (whole_pages) {
        // rows behind the last key are the page's own: what they hold is masked
        const int h = x % TURNS * NH;
        if (h == 0) places(x);
        const char *kb[NH], *vb[NH];
#pragma unroll
        for (int s = 0; s < NH; ++s) {
          kb[s] = lane_ptr(kat, h + s);
          vb[s] = lane_ptr(vat, h + s);
          if (!((good >> (h + s)) & 1)) mask &= ~(0xffffu << 16 * s);
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int r = i * RI + lane / NC, c = lane % NC;
          dma16<ONCE>(lds + i * 1024, kb[i * RI / 16], (uint32_t)((r & 15) * (int)a.pages.k_ts + kchunk(r, c)));
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int r = i * RI + lane / NC, c = lane % NC;
          dma16<ONCE>(lds + KV + i * 1024, vb[i * RI / 16], (uint32_t)((r & 15) * (int)a.pages.v_ts + vchunk(r, c)));
        }
        if constexpr (Q8) {
          const int i0 = __builtin_amdgcn_readlane(at_id, h), i1 = __builtin_amdgcn_readlane(at_id, h + 1);
          const int n0 = __builtin_amdgcn_readlane(at_in, h), n1 = __builtin_amdgcn_readlane(at_in, h + 1);
          dma1(lds + 2 * KV, sbase + (lane & 16 ? i1 : i0) * sps + ((lane & 16 ? n1 : n0) + l16));
        }
      } else {
        int64_t in;
        auto page_of = [&](int r) __attribute__((always_inline)) {   // of row r, -1 outside the cache, and its place
          const int key = min(k0 + r, k_end - 1), p = fdiv(key, a.pages.page), id = table[p];
          in = key - p * a.pages.page.d;
          return (unsigned)id < (unsigned)a.pages.num_pages ? id : -1;
        };
        const int64_t mine = page_of(lane & (KT - 1));
        mask &= (uint32_t)__ballot(mine >= 0);
        const uint8_t* sc = Q8 ? sbase + max(mine, (int64_t)0) * sps + in : nullptr;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int r = i * RI + lane / NC, c = lane % NC;
          const int64_t id = max(page_of(r), 0);
          dma16<ONCE>(lds + i * 1024, kbase + id * a.pages.k_ps + in * a.pages.k_ts + kchunk(r, c));
          dma16<ONCE>(lds + KV + i * 1024, vbase + id * a.pages.v_ps + in * a.pages.v_ts + vchunk(r, c));
        }
        if constexpr (Q8) dma1(lds + 2 * KV, sc);
      }
      return mask;
    };
    // x is a multiple of RING plus the constant i: live[] stays in registers
    auto turn = [&](int x, int i) __attribute__((always_inline)) {
      if (x + RING - 2 < turns) dma_wait<(RING - 2) * (2 * NL + (Q8 ? 1 : 0))>();
      else dma_wait<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the turn before has been read
      char* tile = ring + i * TURN;
      const uint32_t mask = live[i];
      if (x + RING - 1 < turns) {
        live[(i + RING - 1) % RING] = fetch(x + RING - 1);
      }
      const int k0 = k_beg + (x * NW + wave) * KT;
      const bool edge = k0 + KT - 1 > kfirst;   // some row's keys end before the turn's last
      if (mask != ALL) {
        // V rows that are no keys, and their scales, to 0: their probability is 0, their memory anything
#pragma unroll
        for (int z = 0; z < NL; ++z)
          if (!((mask >> (z * RI + lane / NC)) & 1))
            *reinterpret_cast<u32x4*>(tile + KV + (z * 64 + lane) * 16) = u32x4{0, 0, 0, 0};
        if (Q8 && lane >= 32 && !((mask >> (lane - 32)) & 1)) *reinterpret_cast<uint32_t*>(tile + 2 * KV + 4 * lane) = 0;
      }
      if constexpr (Q8) {
        if (edge && kfirst < keys - 1) {
          // nor may a NaN spoil the rows that do not attend it: they are brought to those that do below
#pragma unroll
          for (int z = 0; z < NL; ++z) {
            uint32_t* p = reinterpret_cast<uint32_t*>(tile + KV + (z * 64 + lane) * 16);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t v = p[y], n = nan_bytes(v);
              if (n) {
                p[y] = v & ~n;
                bad = true;
              }
            }
          }
        }
      }
      f32x4 st[NH];
      float vsc[4 * NH];                    // V's scales
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (Q8) {
          const u32x4 ks = *reinterpret_cast<const u32x4*>(tile + 2 * KV + 64 * t + 16 * q4);
          const u32x4 vs = *reinterpret_cast<const u32x4*>(tile + 2 * KV + 128 + 64 * t + 16 * q4);
#pragma unroll
          for (int p = 0; p < NS / 2; ++p) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(tile + 16 * t * D + ko[p]);
            st[t] = El<T>::mma16(from_e4m3<T>(u32x2{y[0], y[1]}, 1.f), qf[2 * p], st[t]);
            st[t] = El<T>::mma16(from_e4m3<T>(u32x2{y[2], y[3]}, 1.f), qf[2 * p + 1], st[t]);
          }
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            st[t][z] *= scale_of(ks[z]);
            vsc[4 * t + z] = scale_of(vs[z]);
          }
        } else {
#pragma unroll
          for (int s = 0; s < NS; ++s) st[t] = El<T>::mma16(*reinterpret_cast<const v8*>(tile + ko[s]), qf[s], st[t]);
        }
      }
      if (mask != ALL) {
#pragma unroll
        for (int z = 0; z < 4 * NH; ++z)
          if (!((mask >> (16 * (z >> 2) + 4 * q4 + (z & 3))) & 1)) st[z >> 2][z & 3] = NEG_INF;
      }
      if (edge) {
#pragma unroll
        for (int z = 0; z < 4 * NH; ++z)
          if (k0 + 16 * (z >> 2) + 4 * q4 + (z & 3) > klast) st[z >> 2][z & 3] = NEG_INF;
      }
      float mx = NEG_INF;
#pragma unroll
      for (int z = 0; z < 4 * NH; ++z) mx = fmaxf(mx, st[z >> 2][z & 3]);
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
      if constexpr (Q8) {
        bf16x8 pf, pr;                      // P times V's scales, and what its rounding leaves
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          const float p = __builtin_amdgcn_exp2f(st[z >> 2][z & 3] * a.c - mc);
          l += p;
          const float y = p * vsc[z];
          pf[z] = (bf16)y;
          pr[z] = (bf16)(y - (float)pf[z]);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const bf16x8 v = from_e4m3<bf16>(tr8(tile + vo[d]), 1.f);
          acc[d] = mfma16(v, pr, mfma16(v, pf, acc[d]));
        }
      } else {
        v4 pf, pr;
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float p = __builtin_amdgcn_exp2f(st[0][z] * a.c - mc);
          l += p;
          pf[z] = (T)p;
          pr[z] = (T)(p - (float)pf[z]);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const v4 v = tr4<T>(reinterpret_cast<const T*>(tile + vo[d]));
          acc[d] = El<T>::mma16k16(v, pr, El<T>::mma16k16(v, pf, acc[d]));
        }
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
    if (bad) s_bad = share;

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
    const bool whole = k_beg == 0 && k_end == keys, spoiled = Q8 && s_bad == share;
    const int piece = u_beg < bfirst ? 1 : 0;
    const int64_t slot = (SHARES && whole ? own_slot(a, e_now, x, b) : (int64_t)w * 2 + piece) * a.HKV + kvh;
    float* pp = a.part + slot * 16 * D;
    float* pm = a.part + a.slots * a.HKV * 16 * D + slot * 32;
    for (int i = tid; i < nrows * (D / 4); i += 64 * NW) {
      const int g = i / (D / 4), d = 4 * (i % (D / 4));
      const int r = 16 * b + g, t = fdiv(r, a.G);
      float mm = NEG_INF, ll = 0.f;
      for (int y = 0; y < NW; ++y) mm = fmaxf(mm, s_ml[y][g][0]);
      const float ref = mm == NEG_INF ? 0.f : mm;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int y = 0; y < NW; ++y) {
        const float f = __builtin_amdgcn_exp2f(s_ml[y][g][0] - ref);
        ll += f * s_ml[y][g][1];
        o += f * *reinterpret_cast<const f32x4*>(ob + (y * 16 + g) * D + d);
      }
      if (spoiled) {
        // the NaN taken out at the edge, to the rows that attend them
        for (int j = max(k_beg, kfirst - KT + 2); j < min(k_end, keys - x.tokens + t + 1); ++j) {
          const int p = fdiv(j, a.pages.page), id = table[p];
          if ((unsigned)id >= (unsigned)a.pages.num_pages) continue;
          const uint32_t v = *reinterpret_cast<const uint32_t*>(vbase + id * a.pages.v_ps +
                                                                (int64_t)(j - p * a.pages.page.d) * a.pages.v_ts + d);
#pragma unroll
          for (int z = 0; z < 4; ++z) o[z] += nan8(v >> (8 * z)) ? __builtin_nanf("") : 0.f;
        }
      }
      if (whole && !SHARES) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        v4 y;
#pragma unroll
        for (int z = 0; z < 4; ++z) y[z] = (T)(o[z] * inv);
        *reinterpret_cast<v4*>(a.o + (int64_t)(x.bos + t) * a.o_ts + (int64_t)(kvh * G + r - t * G) * a.o_hs + 2 * d) = y;
      } else {
        *reinterpret_cast<f32x4*>(pp + g * D + d) = o;
        if (d == 0) {
          pm[2 * g] = mm;
          pm[2 * g + 1] = ll;
        }
      }
    }
    __syncthreads();
  }
}

// Turns of a wave's ring: 64 KB of LDS for the four waves, so that two workgroups fit; three
// beside the tiles of head size 64, of which three workgroups fit.
template <int D> constexpr int ring() { return D == 128 ? 2 : 4; }

template <typename T, int D, bool Q8, bool SHARES>
__global__ __launch_bounds__(64 * NW, OCC) void attn_rows_kernel(Args a) {
  __shared__ __align__(1024) char smem[Shared<D, Q8, ring<D>()>::BYTES];
  __shared__ Shared<D, Q8, ring<D>()> shared;
  attn_rows<T, D, Q8, SHARES, ring<D>()>(a, smem, shared, blockIdx.x);
}

// Many rows behind prefixes in tiles, and the sequences' own keys, in one launch: the first are
// bound by the matrix cores, the second by memory, and workgroups of both kinds, as many of one
// and of the other in turn as there are compute units, run at once (256 sequences to 1031 keys
// behind two prefixes to 16384, 32 / 8 heads of 128: 195 -> 190 us, in 8 bits 181 -> 162, with
// eight of each in turn the first; 138 to 19 keys behind two of 666 28.4 -> 30.6).
constexpr int IN_TURN = 256;
template <typename T, int D, bool Q8>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : 2) void attn_shared_kernel(Args a, FwdArgs f, int tiles, int blocks) {
  constexpr int RING = D == 128 ? 2 : 3;
  constexpr int BYTES = tile_bytes<D, Q8>() > Shared<D, Q8, RING>::BYTES ? tile_bytes<D, Q8>() : Shared<D, Q8, RING>::BYTES;
  __shared__ __align__(1024) char smem[BYTES];
  __shared__ Shared<D, Q8, RING> shared;
  __shared__ int s_bad, s_skip[4];
  const int both = 2 * min((tiles + IN_TURN - 1) / IN_TURN, (blocks + IN_TURN - 1) / IN_TURN), at = blockIdx.x / IN_TURN;
  const bool tile = at < both ? !(at & 1) : tiles > blocks;
  const int i = (at < both ? at >> 1 : at - (both >> 1)) * IN_TURN + blockIdx.x % IN_TURN;
  if (!tile) {
    if (i < blocks) attn_rows<T, D, Q8, true, RING>(a, smem, shared, i);
    return;
  }
  if (i >= tiles) return;
  {
    constexpr bool PAGED = true, PREFIX = true;
    const FwdArgs& a = f;
    const unsigned block = i, blocks = tiles;
#include "attn_tile_body.hpp"
  }
}

// Shares joined: sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s, of the workers that a row's block
// is cut over and (SHARES) of its prefix, whose shares lie here too or, of many rows, in `pre`.
// A workgroup takes RP heads of one token; its threads take a row's shares in turn, D / 4 to a
// share, and meet in LDS.  A row whose block is not cut has been stored.
template <typename T, int D, bool SHARES, int RP>
__global__ __launch_bounds__(256) void attn_rows_join_kernel(Args a, PrefixShares pre) {
  constexpr int TPS = D / 4, SH = 256 / TPS / RP;   // threads of a share, shares of a row at a time
  __shared__ int64_t s_sum[3][4];
  __shared__ int s_entry[2];
  __shared__ __align__(16) f32x4 s_o[SH][RP][TPS];
  __shared__ float s_ml[SH][RP][2];
  const int H = a.HKV * a.G.d, hb = (H + RP - 1) / RP, t = blockIdx.x / hb;
  const int tid = threadIdx.x, lane = tid & 63;
  const int d = tid % TPS, sh = tid / TPS % SH, rp = tid / (TPS * SH);
  const int head = (blockIdx.x - t * hb) * RP + rp;
  const bool here = head < H;
  const int kvh = min(head, H - 1) / a.G.d, g = min(head, H - 1) - kvh * a.G.d;
  // the entries that hold token t, a prefix and a sequence, and what lies before them and in all
  if (tid < 2) s_entry[tid] = -1;
  __syncthreads();
  int64_t sum[3] = {0, 0, 0};               // before the prefix, before the sequence, all
  for (int y = tid; y < a.M + a.N; y += 256) {
    const Entry x = entry_of(a, y);
    const int64_t u = work_of(a, x);
    const bool in = t >= x.bos && t < x.bos + x.tokens;
    sum[2] += u;
    if (in) s_entry[y < a.M ? 0 : 1] = y;
    if (!in && x.bos <= t && y < a.M) sum[0] += u;
    if (y < a.M || (!in && x.bos <= t)) sum[1] += u;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    for (int z = 32; z >= 1; z >>= 1) sum[i] += __shfl_xor(sum[i], z, 64);
    if (lane == 0) s_sum[i][tid >> 6] = sum[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) sum[i] = s_sum[i][0] + s_sum[i][1] + s_sum[i][2] + s_sum[i][3];
  const int64_t stats = a.slots * a.HKV * 16 * D, per = units_per(a, sum[2]);
  float m = NEG_INF, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float* row, const float* ml) __attribute__((always_inline)) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(row + 4 * d);
    const float mn = fmaxf(m, ml[0]), ref = mn == NEG_INF ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(ml[0] - ref);
    l = l * f + ml[1] * e;
    o = o * f + x * e;
    m = mn;
  };
  bool store = SHARES;
#pragma unroll
  for (int i = SHARES ? 0 : 1; i < 2; ++i) {
    const int e = s_entry[i];
    if (e < 0) continue;                    // a row of no sequence, or behind no prefix
    const Entry x = entry_of(a, e);
    const int units = units_of(x), r = (t - x.bos) * a.G.d + g, b = r >> 4;
    if (units == 0) continue;
    const int64_t bfirst = sum[i] + (int64_t)b * (units + SETUP);
    const int64_t w0 = (bfirst + SETUP) / per, w1 = (bfirst + SETUP + units - 1) / per;
    if (!SHARES && w0 == w1) continue;      // stored
    store = true;
#pragma unroll 4
    for (int64_t w = w0 + sh; w <= w1; w += SH) {
      const int64_t at = SHARES && w0 == w1 ? own_slot(a, e, x, b) : w * 2 + (w * per < bfirst ? 1 : 0);
      const int64_t slot = at * a.HKV + kvh;
      add(a.part + (slot * 16 + (r & 15)) * D, a.part + stats + slot * 32 + 2 * (r & 15));
    }
  }
  if constexpr (SHARES) {
    const int64_t r = (int64_t)t * H + min(head, H - 1);
    const float* pstats = pre.part + (int64_t)pre.splits * pre.rows * D;
    for (int s = sh; s < pre.splits; s += SH) {
      const float* ml = pstats + ((int64_t)s * pre.rows + r) * 2;
      if (__builtin_bit_cast(uint32_t, pstats[2 * r]) == NO_SHARE || __builtin_bit_cast(uint32_t, ml[0]) == NO_SHARE) break;
      add(pre.part + ((int64_t)s * pre.rows + r) * D, ml);
    }
  }
  if constexpr (SH > 1) {
    s_o[sh][rp][d] = o;
    if (d == 0) {
      s_ml[sh][rp][0] = m;
      s_ml[sh][rp][1] = l;
    }
    __syncthreads();
  }
  if (sh == 0 && store && here) {
    for (int i = 1; i < SH; ++i) {
      const float mi = s_ml[i][rp][0], mn = fmaxf(m, mi), ref = mn == NEG_INF ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(mi - ref);
      l = l * f + s_ml[i][rp][1] * e;
      o = o * f + s_o[i][rp][d] * e;
      m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typename El<T>::v4 y;
#pragma unroll
    for (int z = 0; z < 4; ++z) y[z] = (T)(o[z] * inv);
    *reinterpret_cast<typename El<T>::v4*>(a.o + (int64_t)t * a.o_ts + (int64_t)head * a.o_hs + 8 * d) = y;
  }
}

// Workers of a kv head: as many as run at once, and no more than `most` units give MIN_UNITS to.
static int64_t workers(int64_t HKV, int64_t most, int per_cu = OCC) {
  int64_t w = (int64_t)per_cu * cu_count() / HKV;
  const int64_t need = (most + MIN_UNITS - 1) / MIN_UNITS;
  if (w > need) w = need;
  return w < 1 ? 1 : w;
}
static int64_t units_at_most(int64_t blocks, int64_t max_keys) { return blocks * ((max_keys + UNIT - 1) / UNIT + SETUP); }
static size_t share_bytes(int64_t slots, int64_t HKV, int32_t D) { return (size_t)(slots * HKV * 16 * (D + 2)) * sizeof(float); }
static size_t prefix_bytes(int64_t splits, int64_t rows, int32_t D) { return (size_t)(splits * rows * (D + 2)) * sizeof(float); }

// Tokens of N sequences, T in all: whole sequences where their tables are short.
static int64_t workers_of(int64_t N, int64_t T, int64_t G, int64_t HKV, int64_t max_keys) {
  return max_keys <= SHORT_KEYS ? 0 : workers(HKV, units_at_most(T * G / 16 + N, max_keys));
}

template <typename T, int D, bool Q8, bool SHARES>
static void launch(const Args& a, const FwdArgs* f, const PrefixShares& pre, hipStream_t s) {
  const int blocks = a.HKV * a.blocks;
  if constexpr (SHARES) {
    if (f) {
      const int tiles = (int)(fwd_blocks(*f) * a.HKV);
      const dim3 grid((unsigned)(IN_TURN * ((tiles + IN_TURN - 1) / IN_TURN + (blocks + IN_TURN - 1) / IN_TURN)));
      hipLaunchKernelGGL((attn_shared_kernel<T, D, Q8>), grid, dim3(64 * NW), 0, s, a, *f, tiles, blocks);
    }
  }
  if (!f) hipLaunchKernelGGL((attn_rows_kernel<T, D, Q8, SHARES>), dim3((unsigned)blocks), dim3(64 * NW), 0, s, a);
  if (!SHARES && a.W <= 1) return;
  const int64_t H = a.HKV * a.G.d, rows = H * a.T;
  // eight rows a workgroup, which finds their entries once, where that leaves enough workgroups
  if (rows >= 1024)
    hipLaunchKernelGGL((attn_rows_join_kernel<T, D, SHARES, 8>), dim3((unsigned)((H + 7) / 8 * a.T)), dim3(256), 0, s, a, pre);
  else
    hipLaunchKernelGGL((attn_rows_join_kernel<T, D, SHARES, 1>), dim3((unsigned)rows), dim3(256), 0, s, a, pre);
}
template <bool Q8, bool SHARES>
static void launch_types(const Args& a, int32_t dtype, int32_t D, hipStream_t s, const FwdArgs* f = nullptr,
                         const PrefixShares& pre = PrefixShares{}) {
  if (dtype == HMX_BF16) {
    if (D == 64) launch<bf16, 64, Q8, SHARES>(a, f, pre, s);
    else launch<bf16, 128, Q8, SHARES>(a, f, pre, s);
  } else {
    if (D == 64) launch<f16, 64, Q8, SHARES>(a, f, pre, s);
    else launch<f16, 128, Q8, SHARES>(a, f, pre, s);
  }
}

// The rows of N sequences, one token each, over the M prefixes that they share, in tiles.  Of
// the two workgroups of a compute unit one takes tiles and one the sequences' own keys, so that
// all run at once (256 sequences to 1031 keys behind two prefixes to 16384: 190 us, with twice as
// many tiles 205, with twice as many workers 200).
static Splits tile_splits(int64_t M, int64_t N, int64_t G, int HKV, int64_t max_prefix, bool packed) {
  const int32_t some = 0;
  const int64_t slots = tile_slots<BM>(packed ? &some : nullptr, M, N, G);
  return splits(packed ? slots - 2 : slots, HKV, max_prefix, 4, 1);
}
// splits whose shares there is room for, with offsets or without
static int64_t tile_splits_most(int64_t M, int64_t N, int64_t G, int HKV, int64_t max_prefix) {
  const int64_t a = tile_splits(M, N, G, HKV, max_prefix, true).most;
  const int64_t b = M == 1 ? tile_splits(M, N, G, HKV, max_prefix, false).most : 1;
  return a > b ? a : b;
}

// What the entry points check alike.
static int check(const char* what, const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t dtype,
                 void* o, int64_t o_token_stride, int64_t o_head_stride, const hmx_paged_kv* cache,
                 const hmx_kv_scales* scales, int32_t N, int32_t H, int32_t HKV, int32_t D, float scale, Args* out) {
  HMX_REQUIRE(D == 64 || D == 128, HMX_EUNSUPPORTED, "%s: head size %d not in {64, 128}", what, D);
  HMX_REQUIRE(dtype == HMX_BF16 || dtype == HMX_F16, HMX_EUNSUPPORTED, "%s: dtype code %d (bf16 or fp16)", what, dtype);
  HMX_REQUIRE(N >= 0 && HKV > 0 && H > 0 && H % HKV == 0, HMX_EINVAL, "%s: N=%d H=%d HKV=%d", what, N, H, HKV);
  HMX_REQUIRE(scale > 0.f && scale < __builtin_inff(), HMX_EINVAL, "%s: scale %g must be positive", what, (double)scale);
  HMX_REQUIRE(cache && cache->num_pages >= 0 && cache->page_size > 0 && cache->table_width >= 0, HMX_EINVAL,
              "%s: cache", what);
  if (N == 0) return HMX_OK;
  HMX_REQUIRE(q && o && cache->seq_lens && has_pages(*cache) && has_scales(*cache, scales), HMX_EINVAL,
              "%s: null pointer", what);
  const int64_t max_keys = (int64_t)cache->table_width * cache->page_size;
  HMX_REQUIRE(max_keys < (1ll << 31) - 256, HMX_EUNSUPPORTED, "%s: a table row holds %lld keys", what,
              (long long)max_keys);
  const int64_t st = q_token_stride | q_head_stride | o_token_stride | o_head_stride;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)o;
  HMX_REQUIRE(st % 8 == 0 && al % 16 == 0 && aligned_pages(*cache, scales != nullptr), HMX_EINVAL,
              "%s: strides must be multiples of 8 elements (a cache's of 16 bytes) and pointers 16-byte aligned", what);
  HMX_REQUIRE(near_rows(cache->k_token_stride) && near_rows(cache->v_token_stride), HMX_EUNSUPPORTED,
              "%s: token strides of the cache past 2^25 elements", what);
  HMX_REQUIRE((int64_t)N * H < (1ll << 30), HMX_EUNSUPPORTED, "%s: %d sequences of %d heads", what, N, H);
  Args& a = *out;
  a.q = (const char*)q; a.o = (char*)o;
  a.q_ts = 2 * q_token_stride; a.q_hs = 2 * q_head_stride;
  a.o_ts = 2 * o_token_stride; a.o_hs = 2 * o_head_stride;
  a.pages = make_pages(*cache, scales);
  a.N = N; a.T = N; a.HKV = HKV; a.G = fast_div(H / HKV);
  a.c = scale * LOG2E;
  return HMX_OK;
}

}  // namespace rows

bool few_rows(int64_t N, int64_t T, int64_t G) { return N > 0 && T * G <= 16 * N; }

size_t few_rows_workspace_bytes(int64_t N, int64_t T, int32_t H, int32_t HKV, int32_t D, int64_t max_keys) {
  const int64_t w = rows::workers_of(N, T, H / HKV, HKV, max_keys);
  return w <= 1 ? 0 : rows::share_bytes(2 * w, HKV, D);
}

void launch_few_rows(const FewRows& f, hipStream_t s) {
  rows::Args a{};
  a.q = (const char*)f.q; a.o = (char*)f.o;
  a.q_ts = 2 * f.q_ts; a.q_hs = 2 * f.q_hs; a.o_ts = 2 * f.o_ts; a.o_hs = 2 * f.o_hs;
  a.pages = f.pages; a.cu = f.cu;
  a.N = f.N; a.T = f.T; a.HKV = f.HKV; a.G = fast_div(f.H / f.HKV);
  a.W = (int32_t)rows::workers_of(f.N, f.T, a.G.d, f.HKV, f.max_keys);
  a.blocks = a.W ? a.W : (int32_t)((int64_t)f.T * a.G.d / 16 + f.N);   // (at most)
  a.c = f.scale * LOG2E; a.fill = f.fill;
  a.part = f.workspace; a.slots = 2ll * a.W;
  rows::launch_types<true, false>(a, f.dtype, f.D, s);
}

}  // namespace attn
}  // namespace hmx

using namespace hmx;

extern "C" int hmx_paged_attention_decode8(const void* q, int64_t q_token_stride,
                                           int64_t q_head_stride, int32_t dtype, void* o,
                                           int64_t o_token_stride, int64_t o_head_stride,
                                           const hmx_paged_kv* cache, const hmx_kv_scales* scales,
                                           int32_t N, int32_t H, int32_t HKV, int32_t D, float scale,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "hmx_paged_attention_decode8";
  HMX_REQUIRE(scales, HMX_EINVAL, "%s: no scales", what);
  attn::rows::Args a{};
  const int rc = attn::rows::check(what, q, q_token_stride, q_head_stride, dtype, o, o_token_stride, o_head_stride,
                                   cache, scales, N, H, HKV, D, scale, &a);
  if (rc != HMX_OK || N == 0) return rc;
  const int64_t max_keys = (int64_t)cache->table_width * cache->page_size;
  const size_t need = hmx_paged_attention_decode8_workspace_bytes(N, H, HKV, D, max_keys);
  HMX_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need), HMX_EINVAL,
              "%s: workspace of %zu bytes is too small", what, workspace_bytes);
  a.W = (int32_t)attn::rows::workers_of(N, N, a.G.d, HKV, max_keys);
  a.blocks = a.W ? a.W : N;
  a.slots = 2ll * a.W;
  a.part = static_cast<float*>(workspace);
  attn::rows::launch_types<true, false>(a, dtype, D, (hipStream_t)stream);
  return check_launch(what);
}

extern "C" size_t hmx_paged_attention_decode8_workspace_bytes(int32_t N, int32_t H, int32_t HKV, int32_t D,
                                                              int64_t max_keys) {
  if (N <= 0 || HKV <= 0 || H <= 0 || H % HKV != 0 || max_keys <= 0) return 0;
  return attn::few_rows_workspace_bytes(N, N, H, HKV, D, max_keys);
}

// Rows behind a prefix are few up to half a tile of 128: four blocks then read the prefix, and
// the tile's idle rows cost about as much (32 / 8 heads of 128 in 8 bits: 64 rows behind 16384
// keys 40.5 us, by tiles 42.8, behind 4096 26.9 and 24.4; 96 rows 29.4 and 26.5; 32 rows 21.7
// either way).
static bool few_behind(int64_t N, int64_t M, int64_t G) { return N * G <= 64 * M; }

namespace {
struct SharedPlan {
  bool few;
  int64_t W, slots, splits;
};
SharedPlan shared_plan(int64_t N, int64_t M, int32_t H, int32_t HKV, int64_t max_keys, int64_t max_prefix) {
  const int64_t G = H / HKV, hb = (G + 15) / 16;
  SharedPlan p;
  p.few = few_behind(N, M, G);
  const int64_t pblocks = p.few && M > 0 ? N * G / 16 + M + 2 : 0;
  p.W = attn::rows::workers(HKV, attn::rows::units_at_most(N * hb, max_keys) + attn::rows::units_at_most(pblocks, max_prefix),
                            p.few || M == 0 ? attn::rows::OCC : 1);
  p.slots = 2 * p.W + N * hb + pblocks;
  p.splits = p.few || M == 0 ? 0 : attn::rows::tile_splits_most(M, N, G, HKV, max_prefix);
  return p;
}
}  // namespace

extern "C" size_t hmx_shared_prefix_decode_workspace_bytes(int32_t N, int32_t M, int32_t H, int32_t HKV,
                                                           int32_t D, int64_t max_keys,
                                                           int64_t max_prefix) {
  if (N <= 0 || M < 0 || HKV <= 0 || H <= 0 || H % HKV != 0 || max_keys < 0 || max_prefix < 0) return 0;
  const SharedPlan p = shared_plan(N, M, H, HKV, max_keys, max_prefix);
  return attn::rows::share_bytes(p.slots, HKV, D) + attn::rows::prefix_bytes(p.splits, (int64_t)N * H, D);
}

extern "C" int hmx_shared_prefix_decode(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                        int32_t dtype, void* o, int64_t o_token_stride,
                                        int64_t o_head_stride, const hmx_paged_kv* cache,
                                        const hmx_kv_scales* scales, const int32_t* prefix_table,
                                        int64_t prefix_table_stride, int32_t prefix_table_width,
                                        const int32_t* prefix_lens, const int32_t* cu_prefix, int32_t N,
                                        int32_t M, int32_t H, int32_t HKV, int32_t D, float scale,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "hmx_shared_prefix_decode";
  attn::rows::Args a{};
  const int rc = attn::rows::check(what, q, q_token_stride, q_head_stride, dtype, o, o_token_stride, o_head_stride,
                                   cache, scales, N, H, HKV, D, scale, &a);
  if (rc != HMX_OK) return rc;
  HMX_REQUIRE(M >= 0 && prefix_table_width >= 0 && (cu_prefix || M == 1), HMX_EINVAL,
              "%s: %d prefixes %s offsets, tables of %d pages", what, M, cu_prefix ? "with" : "without",
              prefix_table_width);
  if (N == 0) return HMX_OK;
  hmx_paged_kv far = *cache;
  far.table = prefix_table; far.table_stride = prefix_table_stride; far.table_width = prefix_table_width;
  far.seq_lens = prefix_lens;
  HMX_REQUIRE(M == 0 || (prefix_lens && attn::has_pages(far) && attn::has_scales(far, scales)), HMX_EINVAL,
              "%s: null pointer", what);
  const int64_t max_keys = (int64_t)cache->table_width * cache->page_size;
  const int64_t max_prefix = (int64_t)prefix_table_width * cache->page_size;
  HMX_REQUIRE(max_prefix < (1ll << 31) - 256, HMX_EUNSUPPORTED, "%s: a table row holds %lld keys", what,
              (long long)max_prefix);
  HMX_REQUIRE(((int64_t)N * a.G.d / 128 + M + 2) * HKV < (1ll << 24) && N + (int64_t)M < (1ll << 30), HMX_EUNSUPPORTED,
              "%s: %d sequences of %d heads behind %d prefixes", what, N, H, M);
  HMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                  workspace_bytes >= hmx_shared_prefix_decode_workspace_bytes(N, M, H, HKV, D, max_keys, max_prefix),
              HMX_EINVAL, "%s: workspace of %zu bytes is too small", what, workspace_bytes);
  const SharedPlan plan = shared_plan(N, M, H, HKV, max_keys, max_prefix);
  a.W = a.blocks = (int32_t)plan.W;
  a.slots = plan.slots;
  a.part = static_cast<float*>(workspace);
  const attn::PrefixShares pre{a.part + attn::rows::share_bytes(a.slots, HKV, D) / sizeof(float), (int64_t)N * H,
                               (int32_t)plan.splits};
  hipStream_t s = (hipStream_t)stream;
  attn::FwdArgs f{};
  if (M > 0 && plan.few) {
    a.M = M; a.p_table = prefix_table; a.p_stride = prefix_table_stride; a.p_lens = prefix_lens; a.p_cu = cu_prefix;
    a.p_width = cache->num_pages > 0 ? prefix_table_width : 0;
  } else if (M > 0) {
    f.q = a.q; f.q_ts = a.q_ts; f.q_hs = a.q_hs;
    f.pages = attn::make_pages(far, scales);
    f.seqs = attn::Seqs{cu_prefix, M, N, a.G.d};
    f.G = a.G; f.H = H; f.HKV = HKV;
    f.slots = (int32_t)attn::tile_slots<attn::BM>(cu_prefix, M, N, a.G.d);
    f.split = attn::rows::tile_splits(M, N, a.G.d, HKV, max_prefix, cu_prefix != nullptr);
    f.nsplit = pre.splits;
    f.places = (int32_t)(cu_count() / HKV);
    f.part = pre.part;
    f.c = a.c;
  }
  const attn::FwdArgs* tiles = pre.splits > 0 ? &f : nullptr;
  if (scales) attn::rows::launch_types<true, true>(a, dtype, D, s, tiles, pre);
  else attn::rows::launch_types<false, true>(a, dtype, D, s, tiles, pre);
  return check_launch(what);
}
