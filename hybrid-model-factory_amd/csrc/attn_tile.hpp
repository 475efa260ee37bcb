// What a tile of 128 rows against their keys, contiguous or in pages, is made of: its arguments,
// the splits of the keys and, in attn_tile_body.hpp, its code.  The kernel of attn_prompt.hip is
// that; attn_rows.hip runs it beside work of its own for rows behind a shared prefix.
#pragma once
#include "attn.hpp"

namespace hmx {
namespace attn {

constexpr int BM = 128, BN = 64;
constexpr float NO_MC = -1e30f;

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
// whether a byte of a cache of 8 bits is e4m3's NaN
__device__ __forceinline__ bool nan8(uint32_t x) { return (x & 0x7f) == 0x7f; }
// and of four bytes, 0xff for each that is
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) {
  const uint32_t n = ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return n | (n - (n >> 7));
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
template <typename T, int D, bool PAGED, bool Q8, bool PREFIX>
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
      if constexpr (Q8) {
        const uint32_t b = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(v) + 8 * x + 4 * h);
#pragma unroll
        for (int z = 0; z < 4; ++z) add[x][z] += nan8(b >> (8 * z)) ? __builtin_nanf("") : 0.f;
      } else {
        const u16x4 b = *reinterpret_cast<const u16x4*>(v + 8 * x + 4 * h);
        const v4 f = __builtin_bit_cast(v4, b);
#pragma unroll
        for (int z = 0; z < 4; ++z) add[x][z] += nonfinite<T>(b[z]) ? (float)f[z] : 0.f;
      }
    }
  }
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    if (add[x][0] == 0.f && add[x][1] == 0.f && add[x][2] == 0.f && add[x][3] == 0.f) continue;
    if (PREFIX || a.nsplit > 1) {
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

template <int D, bool Q8> constexpr int tile_bytes() { return 4 * BN * D * 2 + (Q8 ? 2 * 1024 : 0); }
// Splits of the keys, where the row tiles alone leave compute units idle: as many as give each
// about two workgroups (what runs at once).  A split costs its share's trip through memory and
// the joining launch, so it has at least `least` tiles of keys: four over pages, where there
// are few rows, eight over contiguous keys.  A tile of a longer sequence may take twice as many.
// Prompts, without splits and with: 2048 tokens, 8 / 2 heads of 128, 42.5 -> 31.6 us; 4096,
// 4 / 4 of 64, 58 -> 28; 16384, 2 / 1 of 128, 276 -> 175.
inline Splits splits(int64_t tiles, int HKV, int64_t max_keys, int least, int per_cu = 2) {
  const int64_t live = tiles * HKV, want = (int64_t)per_cu * cu_count(), most = max_keys / (least * BN);
  int64_t even = live > 0 ? want / live : 1;
  if (even > most) even = most;
  if (even > 64) even = 64;
  if (even <= 1) return NO_SPLITS;
  return Splits{(int32_t)even, (int32_t)(2 * even < most ? 2 * even : most), (int32_t)(want / HKV), least};
}

// Workgroups of a kv head.
inline int64_t fwd_blocks(const FwdArgs& a) {
  if (a.split.even <= 1) return a.slots;
  return !a.seqs.cu || a.seqs.N > LANE_SEQS ? (int64_t)a.slots * a.split.even : (int64_t)a.slots + a.split.blocks;
}

}  // namespace attn
}  // namespace hmx
