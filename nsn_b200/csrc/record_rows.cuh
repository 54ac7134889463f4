// Rows of a sealed block restored from its record (K codes as paired halves, V codes as
// paired rows, see code_byte_at) and rounded to the cache dtype, as the bridge's
// restore_group(g, dtype) stores them (loop_kv_nb06_codec.py:36-38).
//
// Both code orders put two 16-code streams into the same BITS words: the low halves hold the
// first (stream A), the high halves the second (stream B).  For K, A and B are channels
// 32 g .. +15 and 32 g + 16 .. +31 of one token; for V, channels 16 c .. +15 of tokens 2 j and
// 2 j + 1.  A value is alpha_t * (min_c + scale_c * code): scale * code is exact in fp32 (11 by
// at most 5 bits), so min + scale * code is one fused multiply-add with the reference's
// rounding, and the product with alpha_t rounds once more before the value is rounded to T.
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

// Sixteen codes of stream A (low halves) and of stream B (high halves) of w[BITS].
template <int BITS>
__device__ __forceinline__ void codes16(const uint32_t (&w)[BITS], uint32_t (&a)[16], uint32_t (&b)[16]) {
  constexpr int kWords = (BITS + 1) / 2;
  constexpr uint32_t kMask = (1u << BITS) - 1u;
  uint32_t sa[kWords], sb[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const uint32_t hi = 2 * i + 1 < BITS ? w[2 * i + 1] : 0u;
    sa[i] = __byte_perm(w[2 * i], hi, 0x5410);
    sb[i] = __byte_perm(w[2 * i], hi, 0x7632);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int bit = BITS * i, word = bit >> 5, sh = bit & 31;
    const bool two = sh + BITS > 32 && word + 1 < kWords;
    a[i] = (two ? __funnelshift_r(sa[word], sa[word + 1 < kWords ? word + 1 : word], sh) : sa[word] >> sh) & kMask;
    b[i] = (two ? __funnelshift_r(sb[word], sb[word + 1 < kWords ? word + 1 : word], sh) : sb[word] >> sh) & kMask;
  }
}

template <typename T> __device__ __forceinline__ uint32_t round2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t round2<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
template <> __device__ __forceinline__ uint32_t round2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}

// Eight values of consecutive channels as 16 bytes of T.
template <typename T>
__device__ __forceinline__ uint4 values8(const uint32_t *code, const __half2 *mn, const __half2 *sc, float alpha) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 m = __half22float2(mn[i]), s = __half22float2(sc[i]);
    const float x = __fmaf_rn(s.x, static_cast<float>(code[2 * i]), m.x);
    const float y = __fmaf_rn(s.y, static_cast<float>(code[2 * i + 1]), m.y);
    r[i] = round2<T>(mul_rn(alpha, x), mul_rn(alpha, y));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

}  // namespace rr
}  // namespace nsnkv
