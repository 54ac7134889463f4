// Shared-prefix attention on the tensor cores (tcgen05).
//
// A CTA attends up to 256 rows (two 128-row tiles) of one kv head over a chunk of the prefix,
// a block of 64 tokens at a time:
//   warps 0-3, 4-7   softmax of row tile 0 and 1, one row per thread (first they bring in Q)
//   warps 8-15       restore: a block's codes become its K and V rows in T, in shared memory
//   warp 16          issues the MMAs, one thread
//   warp 17          loads block records (one bulk copy each)
// TMEM (512 columns): two buffers of S per softmax team (64 columns each), O0 | O1.  S of the
// next blocks is computed while a block is in its softmax; P overwrites its S buffer.  With one
// row tile both softmax teams work on it, on alternate blocks, and join their halves at the end.
//
// What bounds it is the restore: 16384 values a block, about four instructions each, whatever
// the rows.  A code is moved to bits 13..22 of a word, and one AND leaves it the subnormal float
// code 2^(p - 149), p its bit (fused multiply-adds take subnormals at full rate).  With
// a = scale 2^(117 - p) and b = min 2^-32, both exact, one fused multiply-add gives
// 2^-32 (min + scale * code): scale * code has at most 16 bits, so this is the sum rounded once,
// as restore_group rounds it, and no result is subnormal (min and scale are multiples of 2^-24).
// alpha 2^32 takes the factor back in the product (alpha is at most 65504 / 1e-12).  a and b are
// laid out once per block and channel.
//
// Measured: 64 rows over 8192 INT3 tokens, GQA 32:8: 35.6 us with the merge (eight blocks per CTA at
// 2400 cycles between a start of 9 k cycles and 8 k of writing partial rows); 8 rows over 131008
// INT5 tokens, GQA 64:8: 156 us (1.24 TB/s of records, 0.52 instructions per cycle and scheduler,
// 4580 a block).  640 threads leave 96 registers each, and some 80 bytes a thread are spilled.
// Blocks of 64 tokens, not 128, leave TMEM for two buffers of S per team and shared memory for
// four restored blocks.
#pragma once

#include "flash_mma.cuh"
#include "record_rows.cuh"
#include "tc05.cuh"

namespace nsnkv {
namespace xtc {

constexpr int kM = 128;
constexpr int kThreads = 640;
constexpr int kStages = 4;  // restored blocks held
constexpr int kStageRow = kDim * 4 + 16;  // a staged output row (bytes)
constexpr int kRowsBytes = kBlock * kDim * 2;  // K or V of one block

// Records in flight: their own slots, and with one row tile the slots that fit the other tile's Q.
template <int BITS> constexpr int kRaw = BITS == 3 ? 3 : 2;
template <int BITS> constexpr int kRawWide = kRaw<BITS> + kM * kDim * 2 / rr::Rec<BITS>::kBytes;

template <int BITS>
struct Smem {  // q and kv also stage two tiles of output rows, or one behind the other team's half
  uint8_t q[2][kM * kDim * 2];
  uint8_t kv[kStages][2][kRowsBytes];  // each [2 halves of 64 channels][64 tokens][128 B swizzled]
  uint8_t raw[kRaw<BITS>][rr::Rec<BITS>::kBytes];
  float2 ab[2][2][kDim];               // [team][K, V][channel]: a, b of the channel's codes
  uint64_t raw_full[kRawWide<BITS>], raw_empty[kRawWide<BITS>], full[kStages], empty[kStages];
  uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2];
  float e_other[kM];  // log-sum-exps of the second half of the blocks
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

template <int I> struct Int { static constexpr int value = I; };

constexpr float kDown = 0x1p-32f, kUp = 0x1p32f;  // see above: directions are held 2^-32 times as large

// Sixteen codes of a stream -> 16 values of T (channels 16 c ..) as two 16-byte chunks.
template <int BITS, typename T>
__device__ __forceinline__ void values16(const uint32_t (&s)[(BITS + 1) / 2], const float4 (&ab)[8], float alpha,
                                         uint4 (&out)[2]) {
  using W = Window<BITS>;
  uint32_t x[W::kCount], r[8];
  windows<BITS>(s, x);
  const float2 al = make_float2(alpha * kUp, alpha * kUp);
  constexpr uint32_t kMask = (1u << BITS) - 1u;
  auto pair = [&](auto I) {
    constexpr int i = decltype(I)::value;
    const float2 v = make_float2(__uint_as_float(x[2 * i / W::kPer] & kMask << W::bit(2 * i)),
                                 __uint_as_float(x[(2 * i + 1) / W::kPer] & kMask << W::bit(2 * i + 1)));
    const float2 d = tc::fma2(make_float2(ab[i].x, ab[i].y), v, make_float2(ab[i].z, ab[i].w));
    const float2 y = tc::mul2(d, al);
    r[i] = rr::round2<T>(y.x, y.y);
  };
  pair(Int<0>{}), pair(Int<1>{}), pair(Int<2>{}), pair(Int<3>{});
  pair(Int<4>{}), pair(Int<5>{}), pair(Int<6>{}), pair(Int<7>{});
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
  const int nrows = static_cast<int>(end - begin) * G;  // rows * hq fits an int
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge may take its place behind this grid
  if (nloc <= 0 || (blockIdx.z % a.pairs) * 2 * kM >= nrows) return;

  if (warp == 16) {
    tc::tmem_alloc(&S.tmem, 512);
  } else if (tid == 0) {
    for (int i = 0; i < kRawWide<BITS>; ++i) {
      mbar_init(&S.raw_full[i], 1);
      mbar_init(&S.raw_empty[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&S.full[i], 1);
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
  const uint32_t kR = static_cast<int>(blockIdx.z % a.pairs) * 2 * kM + kM < nrows ? kRaw<BITS> : kRawWide<BITS>;
  auto raw = [&](uint32_t slot) {
    return slot < kRaw<BITS> ? S.raw[slot] : S.q[1] + (slot - kRaw<BITS>) * R::kBytes;
  };

  // More row tiles than the grid has: the CTA takes every pairs-th pair of the group in turn.
  // Ring positions and parities run on from one to the next.
  uint32_t blocks = 0, pair_n = 0;  // blocks and pairs taken so far
  uint32_t taken[2] = {0, 0};       // blocks that each softmax team has taken so far
  for (int row0 = (blockIdx.z % a.pairs) * 2 * kM; row0 < nrows;
       row0 += a.pairs * 2 * kM, blocks += nloc, ++pair_n) {
    const int tiles = row0 + kM < nrows ? 2 : 1;  // row tiles of this pair
    const bool split = tiles == 1;                // the teams share one tile
    const int team_blocks[2] = {split ? (nloc + 1) / 2 : nloc, split ? nloc / 2 : nloc};
    if (warp < 8) {  // ---- Q, softmax, output
      const int t = warp >> 2;
      const int first = row0 + (split ? 0 : t * kM);
      if (t < tiles) {
        // Q of the tile into its swizzled place: 16 threads per row, eight rows' pieces on their
        // way at a time (a rolled loop: this code runs once, and cold code costs its fetch).
        constexpr uint32_t kExp = Elem<T>::kBf16 ? 0x7F807F80u : 0x7C007C00u, kOne = Elem<T>::kBf16 ? 0x00800080u : 0x04000400u;
        uint32_t bad = 0;
        const int c = tid & 15;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int r0 = 64 * h + ((tid & 127) >> 4);
          uint4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = first + r0 + 8 * i, p = r / G;
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (r < nrows) {
              const int64_t qr = a.row_index ? __ldg(a.row_index + begin + p) : begin + p;
              if (qr >= 0 && qr < a.rows)
                x[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) +
                                                             (qr * a.hq + head * G + (r - p * G)) * kDim) + c);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = r0 + 8 * i;
            // an exponent of all ones (NaN, infinity) carries into the sign's place
            bad |= ((x[i].x & kExp) + kOne) | ((x[i].y & kExp) + kOne) | ((x[i].z & kExp) + kOne) | ((x[i].w & kExp) + kOne);
            *reinterpret_cast<uint4 *>(S.q[t] + (c >> 3) * (kM * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x[i];
          }
        }
        bad &= 0x80008000u;
        if (bad) set_status(a.status, NSNKV_ST_INPUT_NONFINITE);
        tc::fence_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&S.q_full[t]);
      }
      {
        constexpr float kSc = kScale * fm::kLog2e;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp & 3) << 21);
        const uint32_t o_at = lane_base + 256 + 128 * t;
        float m = -INFINITY, base = 0.f, l = 0.f;
        const bool rows_here = first + 32 * (warp & 3) < nrows;
#pragma unroll 1
        for (int j = 0; j < team_blocks[t]; ++j) {
          const uint32_t n = taken[t] + j, s_at = lane_base + 128 * t + 64 * (n & 1);
          if (!rows_here) {  // none of this warp's rows exist: their P may be anything
            tc::spin(&S.s_full[t][n & 1], n >> 1 & 1, &S.failed, a.status);
            if (lane == 0) tc::mbar_arrive(&S.p_full[t][n & 1]);
            continue;
          }
          tc::spin(&S.s_full[t][n & 1], n >> 1 & 1, &S.failed, a.status);
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
                tc::spin(&S.o_done[t], (n - 1) & 1, &S.failed, a.status);  // P.V of the block before
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
        if (team_blocks[t]) tc::spin(&S.o_done[t], (taken[t] + team_blocks[t] - 1) & 1, &S.failed, a.status);
        tc::fence_after();
        const int r = first + (tid & 127), pr = r / G;
        int64_t qr = -1;
        if (r < nrows) qr = a.row_index ? a.row_index[begin + pr] : begin + pr;
        const bool mine = qr >= 0 && qr < a.rows;
        const int64_t at = (blockIdx.x * a.rows + qr) * a.hq + head * G + (r - pr * G);
        // l is 0 where the team had no block and NaN where every score is NaN, though m, a maximum
        // that passes NaN over, is -inf in both
        float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l), e2 = l == 0.f ? -INFINITY : m + log2f(l);
        // Both teams have seen their last P.V: every MMA is done, and Q and the ring are free.  Team
        // 1's half of a shared tile goes to team 0 through them, column by column of all rows;
        // finished rows are staged there and leave in one bulk copy each (rows 16 bytes apart
        // from a multiple of 128, so that a warp's writes fall into different banks).
        float *other = reinterpret_cast<float *>(S.q) + (tid & 127);
        uint8_t *stage = S.q[0] + (split ? 1 : t) * (kM * kStageRow) + (tid & 127) * kStageRow;
        float w = 0.f;
        tc::bar_named(3, 256);
        if (split && t == 0) {
          tc::bar_named(4, 256);
          const float e1 = S.e_other[tid & 127], top = fmaxf(e2, e1), b0 = top == -INFINITY ? 0.f : top;
          const float x0 = e2 == -INFINITY ? 0.f : fm::ex2(e2 - b0), x1 = e1 == -INFINITY ? 0.f : fm::ex2(e1 - b0);
          const float both = x0 + x1, is = both == 0.f ? 0.f : __fdiv_rn(1.f, both);
          inv *= x0 * is;
          w = x1 * is;
          e2 = both == 0.f ? -INFINITY : top + log2f(both);
        }
        if (!split || t == 0 || team_blocks[1]) {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            float o[32];
            tc::ld32(o, o_at + 32 * i);
            tc::wait_ld();
            tc::pin32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
            if (split && t == 1) {
#pragma unroll
              for (int e = 0; e < 32; ++e) other[(32 * i + e) * kM] = o[e];
              continue;
            }
            if (w != 0.f) {  // (NaN passes)
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = fmaf(w, other[(32 * i + e) * kM], o[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4 *>(stage + 128 * i + 16 * e) =
                  make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          if (mine && !(split && t == 1)) {
            tc::fence_async();
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], 512;" ::"l"(a.o_ws + at * kDim),
                         "r"(tc::saddr(stage))
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          }
        }
        tc::fence_before();
        if (split && t == 1) {
          S.e_other[tid & 127] = e2;
          tc::bar_named(4, 256);
        } else if (mine) {
          a.e_ws[at] = e2;
        }
      }
    } else if (warp < 16) {  // ---- restore
      // Two teams of four warps take alternate blocks, so that one works while the other waits
      // for its record, its tables or a free stage.
      const int team = (warp - 8) >> 2, w4 = warp & 3;
      const int g16 = (w4 & 1) * 4 + (lane >> 3), r8 = (w4 >> 1) * 8 + (lane & 7);
      const int ch = tid & 127;                          // this thread's channel of the a, b tables
      const uint32_t sel = g16 & 1 ? 0x7632u : 0x5410u;  // K: this 16-channel stream's halves of the words
      // this thread's codes in a record and rows in a stage: K tokens r8 + 16 e, V tokens 2 r8 + 32 e
      // and 2 r8 + 32 e + 1 (whose swizzle exchanges the two chunks)
      const int k_src = (r8 * 4 * BITS + (g16 >> 1) * BITS) * 4, v_src = R::kHalf + (r8 * 8 + g16) * BITS * 4;
      const int k_dst = chunk_at(r8, 2 * g16), v_dst = kRowsBytes + chunk_at(2 * r8, 2 * g16);
      const float mul = __int_as_float((127 + 117 - Window<BITS>::bit(ch & 15)) << 23);
      const int mine = team ^ (blocks & 1);                 // the first block of this chunk that is the team's
      uint32_t slot = (blocks + mine) % kR, raw_par = (blocks + mine) / kR & 1;
      uint32_t stage = (blocks + mine) % kStages, par = (blocks + mine) / kStages & 1;
      int bad = 0;
#pragma unroll 1
      for (int j = mine; j < nloc; j += 2) {
        const uint8_t *rec = raw(slot);
        tc::spin(&S.raw_full[slot], raw_par, &S.failed, a.status);
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // K, V; channel pairs as (a, a, b, b)
          const uint16_t *half = reinterpret_cast<const uint16_t *>(rec + x * R::kHalf + R::kMin) + ch;
          const float mn = half_bits_to_f(half[0]), sc = half_bits_to_f(half[128]);
          bad |= !isfinite(mn + sc);
          float *dst = reinterpret_cast<float *>(&S.ab[team][x][ch & ~1]) + (ch & 1);
          dst[0] = sc * mul;
          dst[2] = mn * kDown;
        }
        tc::bar_named(1 + team, 128);
        tc::spin(&S.empty[stage], par ^ 1, &S.failed, a.status);
        uint8_t *rows = S.kv[stage][0];
        const float4 *tab = reinterpret_cast<const float4 *>(S.ab[team][0]) + 8 * g16;
        float4 ab[8];
        uint4 out[2];
        uint32_t st[(BITS + 1) / 2], wd[BITS];
#pragma unroll
        for (int i = 0; i < 8; ++i) ab[i] = tab[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t *src = reinterpret_cast<const uint32_t *>(rec + k_src + e * 16 * 16 * BITS);
          const float alpha = reinterpret_cast<const float *>(rec + R::kAlpha)[r8 + 16 * e];
          bad |= !isfinite(alpha);
#pragma unroll
          for (int i = 0; i < BITS; ++i) wd[i] = src[i];
#pragma unroll
          for (int i = 0; i < (BITS + 1) / 2; ++i)
            st[i] = __byte_perm(wd[2 * i], 2 * i + 1 < BITS ? wd[2 * i + 1] : 0u, sel);
          values16<BITS, T>(st, ab, alpha, out);
          *reinterpret_cast<uint4 *>(rows + k_dst + e * 16 * 128) = out[0];
          *reinterpret_cast<uint4 *>(rows + (k_dst ^ 16) + e * 16 * 128) = out[1];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ab[i] = tab[i + kDim / 2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t *src = reinterpret_cast<const uint32_t *>(rec + v_src + e * 16 * 8 * BITS * 4);
          const float2 alpha = reinterpret_cast<const float2 *>(rec + R::kHalf + R::kAlpha)[r8 + 16 * e];
          bad |= !isfinite(alpha.x) || !isfinite(alpha.y);
#pragma unroll
          for (int i = 0; i < BITS; ++i) wd[i] = src[i];
          uint8_t *dst = rows + e * 32 * 128;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int i = 0; i < (BITS + 1) / 2; ++i)
              st[i] = __byte_perm(wd[2 * i], 2 * i + 1 < BITS ? wd[2 * i + 1] : 0u, y ? 0x7632u : 0x5410u);
            values16<BITS, T>(st, ab, y ? alpha.y : alpha.x, out);
            *reinterpret_cast<uint4 *>(dst + (v_dst ^ (16 * y)) + y * 128) = out[0];
            *reinterpret_cast<uint4 *>(dst + (v_dst ^ (16 * (1 - y))) + y * 128) = out[1];
          }
        }
        tc::fence_async();
        tc::bar_named(1 + team, 128);  // the record and the tables have been read, the rows written
        if ((tid & 127) == 0) {
          tc::mbar_arrive(&S.full[stage]);
          tc::mbar_arrive(&S.raw_empty[slot]);
        }
        slot += 2, stage += 2;
        if (slot >= kR) slot -= kR, raw_par ^= 1;  // kR >= 2
        if (stage >= kStages) stage -= kStages, par ^= 1;
      }
      if (bad) set_status(a.status, NSNKV_ST_INPUT_NONFINITE);
    } else if (warp == 16) {  // ---- MMA: every lane runs the loops, one issues
      const bool lead = tc::elect();
      constexpr uint32_t kIdS = tc::instr_desc<T>(kM, kBlock, false), kIdO = tc::instr_desc<T>(kM, kDim, true);
      const uint64_t qd = tc::smem_desc(tc::saddr(S.q[0]), 16, 1024),
                     kd = tc::smem_desc(tc::saddr(S.kv[0][0]), 16, 1024),
                     vd = tc::smem_desc(tc::saddr(S.kv[0][1]), kRowsBytes / 2, 1024);
      uint32_t cs[2] = {taken[0], taken[1]}, cp[2] = {taken[0], taken[1]};  // S and P.V issued per team
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) tc::spin(&S.q_full[t], pair_n & 1, &S.failed, a.status);
      // S of block sj as soon as the block is restored and a team's buffer is free (P.V of its
      // block there is issued), P.V of block pj as soon as its P is there: whichever comes first.
      const int ahead = split ? 3 : 1;
      int sj = 0, pj = 0, pt = 0;  // pt: the team whose P.V of block pj is next
#pragma unroll 1
      for (int idle = 0; pj < nloc;) {
        const uint32_t s_stage = (blocks + sj) % kStages;
        if (sj < nloc && sj <= pj + ahead && tc::test(&S.full[s_stage], (blocks + sj) / kStages & 1)) {
          tc::fence_after();
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (!split || (sj & 1) == t) {
              if (lead) {
                const uint64_t qa = qd + (split ? 0 : t * (kM * kDim * 2 >> 4)),
                               ka = kd + s_stage * (2 * kRowsBytes >> 4);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  tc::mma_ss(tmem + 128 * t + 64 * (cs[t] & 1), qa + (((i >> 2) * (kM * 128) + (i & 3) * 32) >> 4),
                             ka + (((i >> 2) * (kRowsBytes / 2) + (i & 3) * 32) >> 4), kIdS, i > 0);
                tc::commit(&S.s_full[t][cs[t] & 1]);
              }
              ++cs[t];
            }
          ++sj;
          idle = 0;
          continue;
        }
        const int t = split ? pj & 1 : pt;
        const uint32_t c = t ? cp[1] : cp[0];
        if (sj > pj && tc::test(&S.p_full[t][c & 1], c >> 1 & 1)) {
          tc::fence_after();
          const uint32_t stage = (blocks + pj) % kStages;
          const bool last = split || t == 1;  // of the block's P.V
          if (lead) {
            const uint64_t va = vd + stage * (2 * kRowsBytes >> 4);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              tc::mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 64 * (c & 1) + 8 * i, va + i * (2048 >> 4), kIdO,
                         pj > (split ? 1 : 0) || i > 0);
            tc::commit(&S.o_done[t]);
            if (last) tc::commit(&S.empty[stage]);
          }
          if (t) ++cp[1]; else ++cp[0];
          pt = last ? 0 : 1;
          pj += last;
          idle = 0;
          continue;
        }
        if (++idle > 1 << 16) {  // neither came: give up through the bounded wait
          tc::wait_long(&S.p_full[t][c & 1], c >> 1 & 1, &S.failed, a.status);
          if (*static_cast<volatile int32_t *>(&S.failed)) break;
          idle = 0;
        }
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
        tc::spin(&S.raw_empty[slot], (n / kR & 1) ^ 1, &S.failed, a.status);
        if (lead) {
          mbar_expect_tx(&S.raw_full[slot], R::kBytes);
          bulk_g2s(raw(slot), a.records + head * a.rec_head + page * a.rec_page, R::kBytes, &S.raw_full[slot]);
        }
      }
      __syncwarp();
      if (*static_cast<volatile int32_t *>(&S.failed))  // a wait gave up: let the copies in flight land
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    taken[0] += team_blocks[0], taken[1] += team_blocks[1];
    // The next pair reuses O, the Q tiles and, where a row tile had no rows, untouched barriers.
    if (row0 + a.pairs * 2 * kM < nrows) {
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
