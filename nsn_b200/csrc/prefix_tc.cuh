// Shared-prefix attention on the tensor cores (tcgen05).
//
// A CTA attends up to 256 rows (two 128-row tiles) of one kv head over a chunk of the prefix,
// a block of 64 tokens at a time:
//   warps 0-3, 4-7   softmax of row tile 0 and 1, one row per thread (first they bring in Q)
//   warps 8-15       restore: a block's codes become its K and V rows in T, in shared memory
//   warp 16          issues the MMAs, one thread
//   warp 17          loads block records (one bulk copy each)
// TMEM (512 columns): two buffers of S per row tile (64 columns each), O0 | O1.  S of block
// j + 1 is computed while block j is in its softmax; P overwrites its S buffer.
//
// What bounds it is the restore: 16384 values a block, about four instructions each, whatever
// the rows.  A code is moved to bits 13..22 of a word and one AND-OR with the bits of 1.0f makes
// it the float 1 + code 2^(p - 23), p its bit; with a = scale 2^(23 - p) and b = min - a, the
// direction min + scale * code is one fused multiply-add a * (1 + code 2^(p - 23)) + b.  That is
// the separately rounded min + scale * code wherever b is exact, i.e. wherever min's last bit is
// not below 2^-24 of a (true of unit directions: min and scale within a few powers of two);
// elsewhere it is within 2^-24 a of it.  a and b are laid out once per block and channel.
#pragma once

#include "flash_mma.cuh"
#include "record_rows.cuh"
#include "tc05.cuh"

namespace nsnkv {
namespace xtc {

constexpr int kM = 128;
constexpr int kThreads = 640;
constexpr int kStages = 3;
constexpr int kRowsBytes = kBlock * kDim * 2;  // K or V of one block

template <int BITS> constexpr int kRaw = BITS == 3 ? 4 : 3;  // records in flight

template <int BITS>
struct Smem {
  uint8_t q[2][kM * kDim * 2];
  uint8_t kv[kStages][2][kRowsBytes];  // each [2 halves of 64 channels][64 tokens][128 B swizzled]
  uint8_t raw[kRaw<BITS>][rr::Rec<BITS>::kBytes];
  float2 ab[2][2][kDim];               // [block parity][K, V][channel]: a, b of the channel's codes
  uint64_t raw_full[kRaw<BITS>], raw_empty[kRaw<BITS>], full[kStages], empty[kStages];
  uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2];
  uint32_t tmem;
  int32_t failed;
};

// The window of codes g: the codes at bits kPer * BITS * g .. of the stream, moved to bit kAt.
template <int BITS>
struct Window {
  static constexpr int kPer = BITS == 3 ? 3 : 2, kAt = BITS == 3 ? 14 : 13;
  static constexpr int kCount = (16 + kPer - 1) / kPer;
  static __host__ __device__ constexpr int bit(int i) { return kAt + BITS * (i % kPer); }  // of code i in its window
};
template <int BITS>
__device__ __forceinline__ void windows(const uint32_t (&s)[(BITS + 1) / 2], uint32_t (&x)[Window<BITS>::kCount]) {
  using W = Window<BITS>;
  constexpr int kWords = (BITS + 1) / 2;
#pragma unroll
  for (int g = 0; g < W::kCount; ++g) {
    const int sh = W::kPer * BITS * g - W::kAt;  // right shift of the whole stream
    if (sh <= 0) {
      x[g] = s[0] << -sh;
    } else {
      const int w = sh >> 5;
      x[g] = w + 1 < kWords ? __funnelshift_r(s[w], s[w + 1 < kWords ? w + 1 : w], sh & 31) : s[w] >> (sh & 31);
    }
  }
}

// Sixteen codes of a stream -> 16 values of T (channels 16 c ..) as two 16-byte chunks.
template <int BITS, typename T>
__device__ __forceinline__ void values16(const uint32_t (&s)[(BITS + 1) / 2], const float4 (&ab)[8], float alpha,
                                         uint4 (&out)[2]) {
  using W = Window<BITS>;
  uint32_t x[W::kCount], r[8];
  windows<BITS>(s, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 v;
    v.x = __uint_as_float((x[2 * i / W::kPer] & (((1u << BITS) - 1u) << W::bit(2 * i))) | 0x3F800000u);
    v.y = __uint_as_float((x[(2 * i + 1) / W::kPer] & (((1u << BITS) - 1u) << W::bit(2 * i + 1))) | 0x3F800000u);
    const float2 d = tc::fma2(make_float2(ab[i].x, ab[i].y), v, make_float2(ab[i].z, ab[i].w));
    const float2 y = tc::mul2(d, make_float2(alpha, alpha));
    r[i] = rr::round2<T>(y.x, y.y);
  }
  out[0] = make_uint4(r[0], r[1], r[2], r[3]);
  out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// Byte offset of 16-byte chunk c (8 channels) of token row t in a swizzled [2][64][128 B] tile.
__device__ __forceinline__ int chunk_at(int t, int c) {
  return (c >> 3) * (kRowsBytes / 2) + t * 128 + (((c & 7) ^ (t & 7)) << 4);
}

struct Args {
  const void *q;
  const uint8_t *records;
  const int32_t *table, *n_pages, *row_offsets, *row_index;
  float *o_ws, *e_ws;
  int64_t rows, pages, table_stride, rec_head, rec_page;
  int32_t hq, h, max_pages, chunk_pages, pairs;
  int32_t *status;
};

template <int BITS, typename T>
__global__ void __launch_bounds__(kThreads, 1) prefix_tc_kernel(const __grid_constant__ Args a) {
  extern __shared__ uint8_t smem_raw[];
  using R = rr::Rec<BITS>;
  using Sm = Smem<BITS>;
  constexpr int kR = kRaw<BITS>;
  // the swizzle's pattern repeats every 1024 bytes of the shared address
  Sm &S = *reinterpret_cast<Sm *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.y, group = blockIdx.z / a.pairs, G = a.hq / a.h;
  const int np = min(max(a.n_pages ? a.n_pages[group] : a.max_pages, 0), a.max_pages);
  const int p0 = blockIdx.x * a.chunk_pages, nloc = min(a.chunk_pages, np - p0);
  int64_t begin = 0, end = a.rows;
  if (a.row_offsets) {
    begin = min(max(static_cast<int64_t>(a.row_offsets[group]), int64_t{0}), a.rows);
    end = min(max(static_cast<int64_t>(a.row_offsets[group + 1]), begin), a.rows);
  }
  const int64_t nrows = (end - begin) * G;
  if (nloc <= 0 || (blockIdx.z % a.pairs) * int64_t{2 * kM} >= nrows) return;

  if (warp == 16) {
    tc::tmem_alloc(&S.tmem, 512);
  } else if (tid == 0) {
    for (int i = 0; i < kR; ++i) {
      mbar_init(&S.raw_full[i], 1);
      mbar_init(&S.raw_empty[i], 8);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&S.full[i], 8);
      mbar_init(&S.empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&S.q_full[t], 4);
      mbar_init(&S.o_done[t], 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&S.s_full[t][b], 1);
        mbar_init(&S.p_full[t][b], 4);
      }
    }
    S.failed = 0;
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = S.tmem;

  // More row tiles than the grid has: the CTA takes every pairs-th pair of the group in turn.
  // Ring positions and parities run on from one to the next.
  uint32_t blocks = 0, pair_n = 0;  // blocks and pairs taken so far
  for (int64_t row0 = (blockIdx.z % a.pairs) * int64_t{2 * kM}; row0 < nrows;
       row0 += static_cast<int64_t>(a.pairs) * 2 * kM, blocks += nloc, ++pair_n) {
    const int tiles = row0 + kM < nrows ? 2 : 1;  // row tiles of this pair
    if (warp < 8) {  // ---- Q, softmax, output
      const int t = warp >> 2;
      if (t < tiles) {
        const int64_t first = row0 + t * kM;
        // Q of the tile into its swizzled place: 16 threads per row
        int bad = 0;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const int r = i * 8 + ((tid & 127) >> 4), c = tid & 15;
          const int64_t rr_ = first + r;
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (rr_ < nrows) {
            const int64_t pos = begin + rr_ / G;
            const int64_t qr = a.row_index ? a.row_index[pos] : pos;
            if (qr >= 0 && qr < a.rows)
              x = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (qr * a.hq + head * G + rr_ % G) * kDim)[c];
          }
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = Elem<T>::to_f2(w[e]);
            bad |= !isfinite(f.x) || !isfinite(f.y);
          }
          *reinterpret_cast<uint4 *>(S.q[t] + (c >> 3) * (kM * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x;
        }
        if (bad) set_status(a.status, NSNKV_ST_INPUT_NONFINITE);
        tc::fence_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&S.q_full[t]);

        constexpr float kSc = kScale * fm::kLog2e;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp & 3) << 21);
        const uint32_t o_at = lane_base + 256 + 128 * t;
        float m = -INFINITY, base = 0.f, l = 0.f;
#pragma unroll 1
        for (int j = 0; j < nloc; ++j) {
          const uint32_t n = blocks + j, s_at = lane_base + 128 * t + 64 * (n & 1);
          tc::wait(&S.s_full[t][n & 1], n >> 1 & 1, &S.failed, a.status);
          tc::fence_after();
          float s[64];
          auto fetch = [&] {
            tc::ld32(s, s_at);
            tc::ld32(s + 32, s_at + 32);
            tc::wait_ld();
            tc::pin32(s);
            tc::pin32(s + 32);
          };
          // The maximum in use is the first block's until a block's p sums to 2^15 or more; then
          // it is raised and the block taken again (no p overflows fp16 below that).
          auto top = [&] {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 64; i += 8)
#pragma unroll
              for (int c = 0; c < 4; ++c) mx[c] = tc::max3(mx[c], s[i + c], s[i + 4 + c]);
            return kSc * fmaxf(tc::max3(mx[0], mx[1], mx[2]), mx[3]);
          };
          uint32_t *p = reinterpret_cast<uint32_t *>(s);  // P in place: word e over pair e / 2, taken before
          float sum;
#pragma unroll 1
          for (int again = j == 0;; again = 1) {
            fetch();
            if (again) {
              const float m_new = fmaxf(m, top());
              const float c = m_new == -INFINITY ? 1.f : fm::ex2(m - m_new);
              if (j > 0) {
                tc::wait(&S.o_done[t], (n - 1) & 1, &S.failed, a.status);  // P.V of the block before
                tc::fence_after();
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                  float o[16];
                  tc::ld16(o, o_at + 16 * i);
                  tc::wait_ld();
                  tc::pin16(o);
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] *= c;
                  tc::st16(o_at + 16 * i, reinterpret_cast<uint32_t *>(o));
                }
              }
              l *= c;
              m = m_new;
              base = m == -INFINITY ? 0.f : m;
            }
            const float2 sc2 = make_float2(kSc, kSc), nb2 = make_float2(-base, -base);
            float2 sm[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float2 x = tc::fma2(make_float2(s[2 * e], s[2 * e + 1]), sc2, nb2);
              const float2 y = make_float2(fm::ex2(x.x), fm::ex2(x.y));
              sm[e & 1] = tc::add2(sm[e & 1], y);
              p[e] = fm::round_pair<T>(y.x, y.y);
            }
            sm[0] = tc::add2(sm[0], sm[1]);
            sum = sm[0].x + sm[0].y;
            if (again || !__any_sync(0xffffffffu, !(sum < 32768.f))) break;
          }
          l += sum;
          tc::st32(s_at, p);
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&S.p_full[t][n & 1]);
        }
        tc::wait(&S.o_done[t], (blocks + nloc - 1) & 1, &S.failed, a.status);
        tc::fence_after();
        const int64_t r = first + (tid & 127);
        int64_t qr = -1;
        if (r < nrows) {
          const int64_t pos = begin + r / G;
          qr = a.row_index ? a.row_index[pos] : pos;
        }
        const bool mine = qr >= 0 && qr < a.rows;
        const int64_t at = (blockIdx.x * a.rows + qr) * a.hq + head * G + r % G;
        const float inv = m == -INFINITY ? 0.f : __fdiv_rn(1.f, l);
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          float o[32];
          tc::ld32(o, o_at + 32 * i);
          tc::wait_ld();
          tc::pin32(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
          if (mine)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              tc::store32(a.o_ws + at * kDim + 32 * i + 8 * e, reinterpret_cast<uint32_t *>(o) + 8 * e);
        }
        tc::fence_before();
        if (mine) a.e_ws[at] = m == -INFINITY ? -INFINITY : m + log2f(l);
      }
    } else if (warp < 16) {  // ---- restore
      const int w8 = warp - 8, g16 = (w8 & 1) * 4 + (lane >> 3), r8 = (w8 >> 1) * 8 + (lane & 7);
      const int ch = tid & 127, is_v = (tid >> 7) & 1;  // this thread's channel of the a, b tables (tid 256..511)
      const uint32_t sel = g16 & 1 ? 0x7632u : 0x5410u;  // K: this 16-channel stream's halves of the words
      int bad = 0;
#pragma unroll 1
      for (int j = 0; j < nloc; ++j) {
        const uint32_t n = blocks + j, slot = n % kR, stage = n % kStages;
        const uint8_t *rec = S.raw[slot];
        tc::wait(&S.raw_full[slot], n / kR & 1, &S.failed, a.status);
        {
          const uint8_t *half = rec + is_v * R::kHalf;
          const float mn = half_bits_to_f(reinterpret_cast<const uint16_t *>(half + R::kMin)[ch]);
          const float sc = half_bits_to_f(reinterpret_cast<const uint16_t *>(half + R::kScaleAt)[ch]);
          bad |= !isfinite(mn) || !isfinite(sc);
          using W = Window<BITS>;
          const int i = ch & 15, bit = W::kAt + BITS * (i % W::kPer);
          const float x = sc * __int_as_float((127 + 23 - bit) << 23);
          // pairs of channels as (a, a, b, b)
          float *dst = reinterpret_cast<float *>(&S.ab[n & 1][is_v][ch & ~1]) + (ch & 1);
          dst[0] = x;
          dst[2] = mn - x;
        }
        tc::bar_named(1, 256);
        tc::wait(&S.empty[stage], (n / kStages & 1) ^ 1, &S.failed, a.status);
        float4 ab[8];
        uint4 out[2];
        uint32_t st[(BITS + 1) / 2], wd[BITS];
        const float4 *tab = reinterpret_cast<const float4 *>(S.ab[n & 1][0]) + 8 * g16;
#pragma unroll
        for (int i = 0; i < 8; ++i) ab[i] = tab[i];
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {  // K: token r8 + 32 e
          const int t = r8 + 32 * e;
          const uint32_t *src = reinterpret_cast<const uint32_t *>(rec) + t * 4 * BITS + (g16 >> 1) * BITS;
          const float alpha = reinterpret_cast<const float *>(rec + R::kAlpha)[t];
          bad |= !isfinite(alpha);
#pragma unroll
          for (int i = 0; i < BITS; ++i) wd[i] = src[i];
#pragma unroll
          for (int i = 0; i < (BITS + 1) / 2; ++i)
            st[i] = __byte_perm(wd[2 * i], 2 * i + 1 < BITS ? wd[2 * i + 1] : 0u, sel);
          values16<BITS, T>(st, ab, alpha, out);
          *reinterpret_cast<uint4 *>(S.kv[stage][0] + chunk_at(t, 2 * g16)) = out[0];
          *reinterpret_cast<uint4 *>(S.kv[stage][0] + chunk_at(t, 2 * g16 + 1)) = out[1];
        }
        tab = reinterpret_cast<const float4 *>(S.ab[n & 1][1]) + 8 * g16;
#pragma unroll
        for (int i = 0; i < 8; ++i) ab[i] = tab[i];
        {  // V: tokens 2 r8 and 2 r8 + 1
          const uint32_t *src = reinterpret_cast<const uint32_t *>(rec + R::kHalf) + r8 * 8 * BITS + g16 * BITS;
          const float2 alpha = reinterpret_cast<const float2 *>(rec + R::kHalf + R::kAlpha)[r8];
          bad |= !isfinite(alpha.x) || !isfinite(alpha.y);
#pragma unroll
          for (int i = 0; i < BITS; ++i) wd[i] = src[i];
#pragma unroll 1
          for (int e = 0; e < 2; ++e) {
            const int t = 2 * r8 + e;
#pragma unroll
            for (int i = 0; i < (BITS + 1) / 2; ++i)
              st[i] = __byte_perm(wd[2 * i], 2 * i + 1 < BITS ? wd[2 * i + 1] : 0u, e ? 0x7632u : 0x5410u);
            values16<BITS, T>(st, ab, e ? alpha.y : alpha.x, out);
            *reinterpret_cast<uint4 *>(S.kv[stage][1] + chunk_at(t, 2 * g16)) = out[0];
            *reinterpret_cast<uint4 *>(S.kv[stage][1] + chunk_at(t, 2 * g16 + 1)) = out[1];
          }
        }
        tc::fence_async();
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(&S.full[stage]);
          tc::mbar_arrive(&S.raw_empty[slot]);
        }
      }
      if (bad) set_status(a.status, NSNKV_ST_INPUT_NONFINITE);
    } else if (warp == 16) {  // ---- MMA: every lane runs the loops, one issues
      const bool lead = tc::elect();
      constexpr uint32_t kIdS = tc::instr_desc<T>(kM, kBlock, false), kIdO = tc::instr_desc<T>(kM, kDim, true);
      const uint64_t qd = tc::smem_desc(tc::saddr(S.q[0]), 16, 1024),
                     kd = tc::smem_desc(tc::saddr(S.kv[0][0]), 16, 1024),
                     vd = tc::smem_desc(tc::saddr(S.kv[0][1]), kRowsBytes / 2, 1024);
      auto scores = [&](uint32_t n) {  // S of block n for the pair's row tiles
        const uint32_t stage = n % kStages;
        tc::wait(&S.full[stage], n / kStages & 1, &S.failed, a.status);
        tc::fence_after();
#pragma unroll 1
        for (int t = 0; t < tiles; ++t)
          if (lead) {
            const uint64_t qa = qd + t * (kM * kDim * 2 >> 4), ka = kd + stage * (2 * kRowsBytes >> 4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              tc::mma_ss(tmem + 128 * t + 64 * (n & 1), qa + (((i >> 2) * (kM * 128) + (i & 3) * 32) >> 4),
                         ka + (((i >> 2) * (kRowsBytes / 2) + (i & 3) * 32) >> 4), kIdS, i > 0);
            tc::commit(&S.s_full[t][n & 1]);
          }
      };
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) tc::wait(&S.q_full[t], pair_n & 1, &S.failed, a.status);
      scores(blocks);
#pragma unroll 1
      for (int j = 0; j < nloc; ++j) {
        const uint32_t n = blocks + j, stage = n % kStages;
        if (j + 1 < nloc) scores(n + 1);
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) {
          tc::wait(&S.p_full[t][n & 1], n >> 1 & 1, &S.failed, a.status);
          tc::fence_after();
          if (lead) {
            const uint64_t va = vd + stage * (2 * kRowsBytes >> 4);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              tc::mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 64 * (n & 1) + 8 * i, va + i * (2048 >> 4), kIdO,
                         j > 0 || i > 0);
            tc::commit(&S.o_done[t]);
          }
        }
        if (lead) tc::commit(&S.empty[stage]);
      }
      __syncwarp();
    } else if (warp == 17) {  // ---- records
      const int32_t *row = a.table + group * a.table_stride + p0;
      const bool lead = tc::elect();
      int32_t ids = 0;
#pragma unroll 1
      for (int j = 0; j < nloc; ++j) {
        const uint32_t n = blocks + j, slot = n % kR;
        if ((j & 31) == 0) ids = j + lane < nloc ? row[j + lane] : 0;
        int64_t page = __shfl_sync(0xffffffffu, ids, j & 31);
        if (page < 0 || page >= a.pages) {
          if (lead) set_status(a.status, NSNKV_ST_PAGE);
          page = 0;
        }
        tc::wait(&S.raw_empty[slot], (n / kR & 1) ^ 1, &S.failed, a.status);
        if (lead) {
          mbar_expect_tx(&S.raw_full[slot], R::kBytes);
          bulk_g2s(S.raw[slot], a.records + head * a.rec_head + page * a.rec_page, R::kBytes, &S.raw_full[slot]);
        }
      }
      __syncwarp();
      if (*static_cast<volatile int32_t *>(&S.failed))  // a wait gave up: let the copies in flight land
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    // The next pair reuses O, the Q tiles and, where a row tile had no rows, untouched barriers.
    if (row0 + static_cast<int64_t>(a.pairs) * 2 * kM < nrows) {
      tc::fence_before();
      __syncthreads();
      tc::fence_after();
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 16) tc::tmem_release(tmem, 512);
}

}  // namespace xtc
}  // namespace nsnkv
