// Rows of a sealed block restored from its record (K codes as paired halves, V codes as
// paired rows, see code_byte_at) and rounded to the cache dtype, as the bridge's
// restore_group(g, dtype) stores them (loop_kv_nb06_codec.py:36-38).
//
// Both code orders put two 16-code streams into the same BITS words: the low halves hold the
// first (stream A), the high halves the second (stream B).  For K, A and B are channels
// 32 g .. +15 and 32 g + 16 .. +31 of one token; for V, channels 16 c .. +15 of tokens 2 j and
// 2 j + 1.  A value is alpha_t * (min_c + scale_c * code): scale * code is exact in fp32 (11 by
// at most 5 bits), the sum rounds once, the product with alpha_t once more, and the value is
// rounded to T (prefix_tc.cuh has the arithmetic).
#pragma once

#include "nsnkv_common.cuh"

namespace nsnkv {
namespace rr {

// Field offsets inside a record of BITS-bit codes.
template <int BITS>
struct Rec {
  static constexpr int kCodes = kBlock * kDim * BITS / 8;
  static constexpr int kMin = kCodes, kScaleAt = kCodes + 256, kAlpha = kCodes + 512, kHalf = kCodes + 768;
  static constexpr int kBytes = 2 * kHalf;
};

template <typename T> __device__ __forceinline__ uint32_t round2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t round2<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
template <> __device__ __forceinline__ uint32_t round2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}

}  // namespace rr
}  // namespace nsnkv
