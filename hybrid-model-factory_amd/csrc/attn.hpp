// Shared by the attention kernels (attn_prompt.hip, attn_decode.hip, attn_backward.hip):
// element types of the 32x32 MFMAs, the paged cache's addressing, and the mapping of
// workgroups to the row tiles of packed sequences.
#pragma once
#include "mfma.hpp"

namespace hmx {
namespace attn {

// Operand conventions of the 32x32x16 MFMAs (lane l, h = l >> 5, l32 = l & 31):
//   A: row l32, k = 8h..8h+7;  B: column l32, the same k
//   C/D: column l32, rows 8i + 4h + j in register 4i + j
template <typename T> struct El;
template <> struct El<bf16> {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
  static __device__ __forceinline__ f32x16 mma32(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(v8 a, v8 b, f32x4 c) { return mfma16(a, b, c); }
  // 16x16x16: row (column) l & 15, k = 4 (l >> 4) .. + 3, the C layout of a tile
  static __device__ __forceinline__ f32x4 mma16k16(v4 a, v4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c,
                                                     0, 0, 0);
  }
};
template <> struct El<f16> {
  typedef f16x8 v8;
  typedef f16x4 v4;
  static __device__ __forceinline__ f32x16 mma32(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(v8 a, v8 b, f32x4 c) { return mfma16h(a, b, c); }
  static __device__ __forceinline__ f32x4 mma16k16(v4 a, v4 b, f32x4 c) { return mfma16h_k16(a, b, c); }
};

template <typename T>
__device__ __forceinline__ typename El<T>::v8 pack8(float a0, float a1, float a2, float a3,
                                                    float a4, float a5, float a6, float a7) {
  return typename El<T>::v8{(T)a0, (T)a1, (T)a2, (T)a3, (T)a4, (T)a5, (T)a6, (T)a7};
}

// the transposing LDS read of 4 keys of one column (see ld_tr in mfma.hpp): the lane's
// own address, the 16 lanes of a group covering 4 rows x 16 columns
template <typename T>
__device__ __forceinline__ typename El<T>::v4 tr4(const T* p) {
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)(p));
  return __builtin_bit_cast(typename El<T>::v4, r);
}
template <typename T>
__device__ __forceinline__ typename El<T>::v8 join(typename El<T>::v4 a, typename El<T>::v4 b) {
  return typename El<T>::v8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The 16-byte chunk at which chunk c of row r of a tile sits in LDS.  Rows are read 16 at
// a time at one chunk (row fragments) and four at a time over four chunks (the transposing
// reads): the low two bits of the row choose among the groups of four chunks, the next
// bits the place within, so both kinds of read are spread over all banks.
template <int D> __device__ __forceinline__ int swz(int r, int c) {
  return D == 128 ? c ^ (((r & 3) << 2) | ((r >> 2) & 3))
                  : c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

// The element offset, in a tile at a multiple of 16 rows, at which a lane's transposing
// reads of 32 columns (chunks 4 d .. 4 d + 3) and rows 4 h .. 4 h + 3 start; with `up` 8 rows
// on, where the swizzle's second bit is the other one.
template <int D> __device__ __forceinline__ int tr_offset(int lane, int d, bool up) {
  const int s = lane & 15, g = (lane >> 4) & 1, r = 4 * (lane >> 5) + (s >> 2) + (up ? 8 : 0);
  return r * D + swz<D>(r, 4 * d + 2 * g + ((s & 3) >> 1)) * 8 + 4 * (s & 1);
}

// Nothing moves across it: the kernels' inner blocks are written in the order in which they
// are to issue, a few instructions between two fences (loads ahead of their use, vector
// instructions between matrix products); left to itself the scheduler gathers them by kind.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// max and sum over the two halves of a wave, in the VALU
__device__ __forceinline__ float half_max(float a) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a),
                                                  __builtin_bit_cast(unsigned, a), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float q4_max(float a) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a),
                                                  __builtin_bit_cast(unsigned, a), false, false);
  return half_max(fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])));
}

// 16 bytes a lane from memory into LDS without a trip through registers: lane l's go to
// lds + 16 l (uniform, in M0), from base (uniform) + off or from its own address.  The
// compiler does not see the write: a tile is read after dma_wait() and a barrier.  (M0 is
// reserved and cannot be named as clobbered; nothing the compiler emits in these kernels
// keeps a value in it.)
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)(p);
}
__device__ __forceinline__ void dma16(uint32_t lds, const char* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void dma16(uint32_t lds, const char* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(at) : "memory");
}
__device__ __forceinline__ void dma4(uint32_t lds, const char* at) {   // 4 bytes a lane, to lds + 4 l
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :: "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(at) : "memory");
}
template <int N> __device__ __forceinline__ void dma_wait() {   // all but the last N
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
// an int32 at a uniform index of memory that no kernel in flight writes
__device__ __forceinline__ int uniform_load(const int32_t* p, int64_t i) {
  return *((__attribute__((address_space(4))) const int32_t*)(uintptr_t)(p + i));
}
template <typename P> __device__ __forceinline__ P* uniform_ptr(P* p) {
  const uint64_t x = (uint64_t)p;
  return (P*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
              (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

constexpr float NEG_INF = -__builtin_inff();
constexpr float LOG2E = 1.4426950408889634f;

// x / d and x % d for 0 <= x < 2^31 by a 64-bit reciprocal m = ceil(2^64 / d) (0: d = 1):
// x m / 2^64 exceeds x / d by less than x / 2^64 < 1 / d, so the floor is exact
struct FastDiv {
  uint64_t m;
  int32_t d;
};
inline FastDiv fast_div(int32_t d) {
  return FastDiv{d <= 1 ? 0 : ~0ull / (uint64_t)d + 1, d};   // ~0 / d + 1 = ceil(2^64 / d)
}
__device__ __forceinline__ int fdiv(int x, const FastDiv& f) {
  return f.m == 0 ? x : (int)__umul64hi((uint64_t)(uint32_t)x, f.m);
}
// the same for slots of a cache, which may pass 2^31: x d < 2^64 is all it needs
__device__ __forceinline__ int64_t fdiv64(int64_t x, const FastDiv& f) {
  return f.m == 0 ? x : (int64_t)__umul64hi((uint64_t)x, f.m);
}

// ------------------------------------------------------------------ paged cache
struct Pages {
  const char* k;
  const char* v;
  int64_t k_ps, k_ts, k_hs, v_ps, v_ts, v_hs;   // strides in bytes
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  int32_t width, num_pages;
  FastDiv page;
};

// the kernels reach the 16 rows of a load group by 32-bit offsets
inline bool near_rows(int64_t token_stride) { return token_stride >= 0 && token_stride < (1ll << 25); }

// a cache or a table of no pages may be NULL: it holds no keys
inline bool has_pages(const hmx_paged_kv& c) {
  return c.num_pages == 0 || c.table_width == 0 || (c.k && c.v && c.table);
}

inline Pages make_pages(const hmx_paged_kv& c) {
  Pages p;
  p.k = static_cast<const char*>(c.k);
  p.v = static_cast<const char*>(c.v);
  p.k_ps = 2 * c.k_page_stride; p.k_ts = 2 * c.k_token_stride; p.k_hs = 2 * c.k_head_stride;
  p.v_ps = 2 * c.v_page_stride; p.v_ts = 2 * c.v_token_stride; p.v_hs = 2 * c.v_head_stride;
  p.table = c.table; p.table_stride = c.table_stride; p.lens = c.seq_lens;
  p.width = c.num_pages > 0 ? c.table_width : 0;   // an empty cache holds no keys
  p.num_pages = c.num_pages; p.page = fast_div(c.page_size);
  return p;
}

// ------------------------------------------------------------------ packed sequences
// Rows are (token, head of the group), G to a token.  Boundaries b(0) = 0, b(1) = cu[0],
// ..., b(N + 1) = cu[N], b(N + 2) = T cut the tokens into N sequences and the gaps before
// and behind them.  Part e starts at tile slot f(e) = floor(b(e) G / BM) + e: between f(e)
// and f(e + 1) lie at least ceil(rows / BM) slots, so a workgroup finds its tile from its
// slot with a search, without a plan made of the lengths on the host.
struct Seqs {
  const int32_t* cu;   // NULL: N sequences of T / N tokens
  int32_t N, T, G;
};

struct Tile {
  int seq;             // -1: rows of no sequence
  int bos, tokens;     // the part's first token and its tokens
  int row0, rows;      // the tile's first row in the part, the part's rows; row0 >= rows: nothing to do
  int sp, ns;          // the split of its keys, of ns
};

// How the keys of row tiles are split, for kernels whose shares are joined: `even` splits of
// every tile, or, where the sequences' keys are at hand (next_tile), splits of one length, of
// at least `least` key tiles, at most `most` a row tile and `blocks` in all.
struct Splits {
  int32_t even, most, blocks, least;
};
constexpr Splits NO_SPLITS{1, 1, 0, 0};

__device__ __forceinline__ int seq_bound(const Seqs& s, int e) {
  if (e == 0) return 0;
  if (e == s.N + 2) return s.T;
  return min(max(s.cu[e - 1], 0), s.T);
}

template <int BM>
__device__ __forceinline__ Tile find_tile(const Seqs& s, int slot) {
  Tile t;
  t.sp = 0;
  t.ns = 1;
  if (!s.cu) {
    const int len = s.T / s.N, per = (int)(((int64_t)len * s.G + BM - 1) / BM);
    t.seq = slot / max(per, 1);
    t.bos = t.seq * len;
    t.tokens = len;
    t.row0 = (slot - t.seq * per) * BM;
    t.rows = len * s.G;
    if (t.seq >= s.N || per == 0) t.rows = 0;
    return t;
  }
  const int lane = threadIdx.x & 63;
  int lo = 0, span = s.N + 2;
  while (span > 1) {
    const int step = (span + 63) >> 6, e = lo + lane * step;
    const bool in = lane * step < span &&
                    (int64_t)seq_bound(s, min(e, s.N + 2)) * s.G / BM + e <= slot;
    const unsigned long long m = __ballot(in) | 1ull;   // f(0) = 0 <= slot
    const int p = 63 - __builtin_clzll(m);
    span = min(step, span - p * step);
    lo += p * step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  t.bos = seq_bound(s, lo);
  t.tokens = max(seq_bound(s, lo + 1) - t.bos, 0);
  t.seq = (lo == 0 || lo == s.N + 1) ? -1 : lo - 1;
  t.row0 = (int)(slot - ((int64_t)t.bos * s.G / BM + lo)) * BM;
  t.rows = t.tokens * s.G;
  return t;
}

// The tile of the block in place `at`, heaviest first: a row tile's work grows with the keys
// before it, so a sequence's tiles go from the last (LAST) to the first, or from the first
// where the first have most; and of up to LANE_SEQS packed sequences those with most keys come
// first (their lengths are in the lanes of a wave; more go as they lie).  Whatever comes
// last then is short.  Splits of unequal sequences get one length, the work over (blocks -
// tiles): rounded up for every tile they are no more than `blocks`, so all run at once and end
// together.  lens: the sequences' keys, NULL where they are their tokens.
constexpr int LANE_SEQS = 62;
template <int BM, bool LAST>
__device__ __forceinline__ Tile next_tile(const Seqs& s, const int32_t* lens, int at, int slots,
                                          Splits split = NO_SPLITS) {
  if (!s.cu || s.N < 1 || s.N > LANE_SEQS) {
    const int sp = split.even > 1 ? at % split.even : 0;
    if (split.even > 1) at /= split.even;
    Tile t = find_tile<BM>(s, LAST ? slots - 1 - at : at);
    t.sp = sp;
    t.ns = split.even;
    return t;
  }
  const int lane = threadIdx.x & 63, parts = s.N + 2;
  const bool in = lane < parts, gap = lane == 0 || lane == s.N + 1;
  const int bos = in ? seq_bound(s, lane) : 0;
  const int tokens = in ? max(seq_bound(s, lane + 1) - bos, 0) : 0;
  const int tiles = (int)(((int64_t)tokens * s.G + BM - 1) / BM);
  const int keys = gap ? -1 : lens ? lens[min(max(lane - 1, 0), s.N - 1)] : tokens;
  int ns = 1;
  if (split.even > 1) {
    const int kt = gap ? 0 : max(keys, 0) / 64 + 1;
    int64_t work = (int64_t)tiles * kt;
    int all = tiles;
    for (int d = 32; d >= 1; d >>= 1) {
      work += __shfl_xor(work, d, 64);
      all += __shfl_xor(all, d, 64);
    }
    const int over = max(split.blocks - all, 1);
    const int share = (int)max((work + over - 1) / over, (int64_t)split.least);
    ns = min(max((kt + share - 1) / share, 1), split.most);
  }
  const int blocks = tiles * ns;
  int start = 0;                              // blocks of the parts before this lane's
  for (int f = 0; f < parts; ++f) {
    const int k = __builtin_amdgcn_readlane(keys, f), n = __builtin_amdgcn_readlane(blocks, f);
    start += k > keys || (k == keys && f < lane) ? n : 0;
  }
  const unsigned long long m = __ballot(in && at >= start && at < start + blocks);
  Tile t{-1, 0, 0, 0, 0, 0, 1};
  if (m == 0) return t;
  const int e = __builtin_ctzll(m);
  t.seq = e == 0 || e == s.N + 1 ? -1 : e - 1;
  t.bos = __builtin_amdgcn_readlane(bos, e);
  t.tokens = __builtin_amdgcn_readlane(tokens, e);
  int i = at - __builtin_amdgcn_readlane(start, e);
  t.ns = __builtin_amdgcn_readlane(ns, e);
  if (split.even > 1) {
    t.sp = i % t.ns;
    i /= t.ns;
  }
  t.row0 = (LAST ? __builtin_amdgcn_readlane(tiles, e) - 1 - i : i) * BM;
  t.rows = t.tokens * s.G;
  return t;
}

// Where all of a kv head's blocks run at once, two to a compute unit, the block `at` places on
// shares one with block `at`: the second half goes from the lightest up, so that every unit
// gets about the same (8192 tokens, 8 / 2 heads: 174 -> 169 us; 16384, 2 / 1, split: 216 -> 181).
// The blocks are the grid's.  Of packed sequences that counts the slots without a tile too,
// which then lie opposite the heaviest tiles: still better than no pairing (8 prompts, 6000
// tokens, 8 / 4 heads: 38.6 -> 36.2; drafts of 100 sequences 45.7 -> 44.8).  Splits by length
// have more blocks than run at once, and are never paired.
__device__ __forceinline__ int place(int at, int blocks, int places) {
  return at >= places && blocks <= 2 * places ? blocks - 1 - (at - places) : at;
}

template <int BM>
inline int64_t tile_slots(const int32_t* cu, int64_t N, int64_t T, int64_t G) {
  if (!cu) return N * ((T / N * G + BM - 1) / BM);
  return T * G / BM + N + 2;
}

}  // namespace attn
}  // namespace hmx
