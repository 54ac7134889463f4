// Attention of 16 query rows per warp over 64-token K / V tiles in shared memory
// (mma.sync m16n8k16), shared by the prompt and the shared-prefix kernels.
//
// Online softmax: with scores x_j = q.k_j * scale * log2(e), a running maximum m and sum l,
//   m' = max(m, max_j x_j),  p_j = 2^(x_j - m'),  l' = l 2^(m - m') + sum_j p_j,
//   o' = o 2^(m - m') + sum_j p_j v_j,
// so one pass over K and V gives o / l and the log-sum-exp (m + log2 l) ln 2.  m, l and o
// stay in fp32; p_j is rounded to the operand type of the P.V product (2^-12 of its size for
// fp16, 2^-9 for bf16), l sums the unrounded p_j.
#pragma once

#include "nsnkv_common.cuh"

namespace nsnkv {
namespace fm {

constexpr int kTile = 64;            // tokens per tile
constexpr int kRow = kDim + 8;       // shared row stride (elements): 272 B keeps ldmatrix conflict-free
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(row))));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void *row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(row))));
}

template <typename T> __device__ __forceinline__ uint32_t round_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t round_pair<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
template <> __device__ __forceinline__ uint32_t round_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}

// acc + 0 * w per element of a packed pair: NaN once a w held NaN or an infinity, else 0.
template <typename T> __device__ __forceinline__ uint32_t add_zero_times(uint32_t acc, uint32_t w);
template <> __device__ __forceinline__ uint32_t add_zero_times<__half>(uint32_t acc, uint32_t w) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&w), __float2half2_rn(0.f),
                            *reinterpret_cast<const __half2 *>(&acc));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <> __device__ __forceinline__ uint32_t add_zero_times<__nv_bfloat16>(uint32_t acc, uint32_t w) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&w), __float2bfloat162_rn(0.f),
                                   *reinterpret_cast<const __nv_bfloat162 *>(&acc));
  return *reinterpret_cast<const uint32_t *>(&r);
}

// The state of a warp's 16 rows.  Lane (g = lane / 4, t = lane % 4) holds rows g and g + 8.
struct Rows {
  uint32_t q[8][4];  // A fragments of Q, k-step ks: channels 16 ks ..
  float o[16][4];    // accumulators, channel tile nt: channels 8 nt + 2 t, + 1 of rows g, g + 8
  float m[2], l[2];  // l: this lane's share of the row sum

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int nt = 0; nt < 16; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][i] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }

  // Q fragments from two row pointers (null: a row of zeros)
  template <typename T>
  __device__ __forceinline__ void load_q(const T *r0, const T *r1, int lane) {
    const int t = lane & 3;
    const uint32_t *p0 = reinterpret_cast<const uint32_t *>(r0), *p1 = reinterpret_cast<const uint32_t *>(r1);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      q[ks][0] = p0 ? p0[8 * ks + t] : 0u;
      q[ks][1] = p1 ? p1[8 * ks + t] : 0u;
      q[ks][2] = p0 ? p0[8 * ks + 4 + t] : 0u;
      q[ks][3] = p1 ? p1[8 * ks + 4 + t] : 0u;
    }
  }

  // Scores of one tile of 64 tokens into probabilities p (fp32) with the running maximum, sum
  // and accumulators rescaled.  Token j of the tile is seen by row g when j < n0 and by row
  // g + 8 when j < n1.
  template <typename T>
  __device__ __forceinline__ void scores(const uint16_t (*ks)[kRow], int n0, int n1, int lane, float (&s)[8][4]) {
    const int t = lane & 3, lr = lane & 7, lq = lane >> 3;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t b[4];
        ldsm4(b, &ks[8 * nt + lr][32 * kk + 8 * lq]);
        mma16816<T>(s[nt], q[2 * kk][0], q[2 * kk][1], q[2 * kk][2], q[2 * kk][3], b[0], b[1]);
        mma16816<T>(s[nt], q[2 * kk + 1][0], q[2 * kk + 1][1], q[2 * kk + 1][2], q[2 * kk + 1][3], b[2], b[3]);
      }
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = 8 * nt + 2 * t + i;
        s[nt][i] = j < n0 ? s[nt][i] * (kScale * kLog2e) : -INFINITY;
        s[nt][2 + i] = j < n1 ? s[nt][2 + i] * (kScale * kLog2e) : -INFINITY;
        mx0 = fmaxf(mx0, s[nt][i]);
        mx1 = fmaxf(mx1, s[nt][2 + i]);
      }
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
    }
    const float m0 = fmaxf(m[0], mx0), m1 = fmaxf(m[1], mx1);
    // a row that has seen nothing keeps m = -inf; its p must be 0, not NaN
    const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
    const float c0 = ex2(m[0] - b0), c1 = ex2(m[1] - b1);
    m[0] = m0;
    m[1] = m1;
    l[0] *= c0;
    l[1] *= c1;
#pragma unroll
    for (int nt = 0; nt < 16; ++nt) {
      o[nt][0] *= c0;
      o[nt][1] *= c0;
      o[nt][2] *= c1;
      o[nt][3] *= c1;
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      s[nt][0] = ex2(s[nt][0] - b0);
      s[nt][1] = ex2(s[nt][1] - b0);
      s[nt][2] = ex2(s[nt][2] - b1);
      s[nt][3] = ex2(s[nt][3] - b1);
      l[0] += s[nt][0] + s[nt][1];
      l[1] += s[nt][2] + s[nt][3];
    }
  }

  // o += round(p) . V.  GUARD: V rows with a bit in `skip` (token j: bit j) enter as zeros.
  template <typename T, bool GUARD>
  __device__ __forceinline__ void pv(const float (&s)[8][4], const uint16_t (*vs)[kRow], uint64_t skip, int lane) {
    const int t = lane & 3, lr = lane & 7, lq = lane >> 3;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t p[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[2 * e] = round_pair<T>(s[2 * kk + e][0], s[2 * kk + e][1]);
        p[2 * e + 1] = round_pair<T>(s[2 * kk + e][2], s[2 * kk + e][3]);
      }
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if constexpr (GUARD) {  // B fragment rows of this lane: tokens 16 kk + 2 t, + 1 and 8 further
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 16 * kk + 8 * e + 2 * t;
          keep[e] = (skip >> j & 1 ? 0u : 0xffffu) | (skip >> (j + 1) & 1 ? 0u : 0xffff0000u);
        }
      }
#pragma unroll
      for (int nt = 0; nt < 16; nt += 2) {
        uint32_t b[4];
        ldsm4t(b, &vs[16 * kk + 8 * (lq & 1) + lr][8 * nt + 8 * (lq >> 1)]);
        mma16816<T>(o[nt], p[0], p[1], p[2], p[3], b[0] & keep[0], b[1] & keep[1]);
        mma16816<T>(o[nt + 1], p[0], p[1], p[2], p[3], b[2] & keep[0], b[3] & keep[1]);
      }
    }
  }

  // One tile of 64 tokens.
  template <typename T>
  __device__ __forceinline__ void tile(const uint16_t (*ks)[kRow], const uint16_t (*vs)[kRow], int n0, int n1,
                                       int lane) {
    float s[8][4];
    scores<T>(ks, n0, n1, lane, s);
    pv<T, false>(s, vs, 0, lane);
  }

  // One tile some of whose V rows hold NaN or infinities: those rows leave the product and are
  // added to the rows that see their token only.
  template <typename T>
  __device__ __forceinline__ void tile_guarded(const uint16_t (*ks)[kRow], const uint16_t (*vs)[kRow], int n0, int n1,
                                            int lane) {
    float s[8][4];
    scores<T>(ks, n0, n1, lane, s);
    uint64_t skip = 0;
#pragma unroll 1
    for (int j = 0; j < kTile; ++j) {
      int bad = 0;
      for (int c = 2 * lane; c < kDim; c += 64) {
        const float2 x = Elem<T>::to_f2(*reinterpret_cast<const uint32_t *>(&vs[j][c]));
        bad |= !isfinite(x.x) || !isfinite(x.y);
      }
      if (__any_sync(0xffffffffu, bad)) skip |= uint64_t{1} << j;
    }
    pv<T, true>(s, vs, skip, lane);
#pragma unroll
    for (int n8 = 0; n8 < 8; ++n8) {
      uint32_t todo = static_cast<uint32_t>(skip >> (8 * n8)) & 0xffu;
#pragma unroll 1
      while (todo) {
        const int jj = __ffs(todo) - 1, j = 8 * n8 + jj;
        todo &= todo - 1;
        // token j's p of this lane's two rows sits in lane 4 g + jj / 2
        const int from = (lane & ~3) | (jj >> 1);
        const float p0 = __shfl_sync(0xffffffffu, jj & 1 ? s[n8][1] : s[n8][0], from);
        const float p1 = __shfl_sync(0xffffffffu, jj & 1 ? s[n8][3] : s[n8][2], from);
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) {
          const float2 x = Elem<T>::to_f2(*reinterpret_cast<const uint32_t *>(&vs[j][8 * nt + 2 * (lane & 3)]));
          if (j < n0) {
            o[nt][0] += p0 * x.x;
            o[nt][1] += p0 * x.y;
          }
          if (j < n1) {
            o[nt][2] += p1 * x.x;
            o[nt][3] += p1 * x.y;
          }
        }
      }
    }
  }

  // Row sums over the four lanes of a row; inv: 1 / l.  l is 0 for a row that saw nothing (any
  // finite score leaves at least one p near 1) and NaN for one whose scores are all NaN, though m,
  // a maximum that passes NaN over, is -inf in both.
  __device__ __forceinline__ void finish(float (&inv)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      inv[i] = l[i] == 0.f ? 0.f : __fdiv_rn(1.f, l[i]);
    }
  }
  // Log-sum-exp of row i of this lane (base 2), -inf for a row that saw nothing.
  __device__ __forceinline__ float lse2(int i) const { return l[i] == 0.f ? -INFINITY : m[i] + log2f(l[i]); }
};

}  // namespace fm
}  // namespace nsnkv
