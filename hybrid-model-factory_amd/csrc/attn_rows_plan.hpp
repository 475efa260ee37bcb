// Index arithmetic of attn_rows.hip (plain C++, for host and device).
#pragma once
#include <stdint.h>

namespace hmx {
namespace attn {
namespace rows {

// The first key of half `half` (sixteen keys) of turn `turn` of a wave, of NW waves that take KT
// keys in turn from k_beg on; where that lies behind key k_end - 1, that key's own sixteen's
// first.  Turns are asked for far ahead, up to 64 halves of four waves (8192 keys) behind a share
// whose end may be key 2^31 - 257: their keys pass 2^31, but not 2^32.
template <int NW, int KT> constexpr int half_row(int k_beg, int k_end, int turn, int wave, int half) {
  const uint32_t r = (uint32_t)k_beg + ((uint32_t)turn * NW + wave) * KT + 16 * half;
  const uint32_t last = (uint32_t)(k_end - 1) & ~15u;
  return (int)(r < last ? r : last);
}

}  // namespace rows
}  // namespace attn
}  // namespace hmx
