// Prompt attention on the tensor cores (tcgen05), for prompts of a few tiles and more.
//
// A CTA attends 256 query rows of one head (two 128-row tiles) over 128-token K / V tiles:
//   warps 0-3, 4-7   softmax of row tile 0 and 1, one row per thread
//   warp 8           issues the MMAs, one thread
//   warp 9           issues the TMA loads: Q once, K and V through a ring of kStages tiles
// TMEM (512 columns): S0 | S1 | O0 | O1.  Per tile and row tile: S = Q.K^T into S; the
// softmax warps read a row of S into registers, write P = 2^(x - m) in 16 bits over S and the
// tensor core adds P.V to O, P read from TMEM.  While one row tile is in its softmax the
// tensor core works on the other.
//
// The running maximum m is only raised when a row's maximum passed it by more than 8 (in log2
// units): p stays below 2^8, l and O are then in units of the stale maximum, which cancels in
// O / l, and O (in TMEM) is rescaled rarely instead of once per tile.
#pragma once

#include "flash_mma.cuh"
#include "tc05.cuh"

namespace nsnkv {
namespace ptc {

constexpr int kM = 128, kN = 128;  // rows of a row tile, tokens of a K / V tile
constexpr int kStages = 5;
constexpr int kTileBytes = kN * kDim * 2;
constexpr int kThreads = 384;
constexpr float kRaise = 8.f;

struct Smem {
  uint8_t q[2][kTileBytes];        // each [2 halves of 64 channels][128 rows][128 B swizzled]
  uint8_t kv[kStages][kTileBytes];
  uint64_t q_full[2], kv_full[kStages], kv_empty[kStages], s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
  int32_t failed;
  int32_t redo[2];
};

struct Args {
  const int32_t *cu;
  void *out;
  float *lse;
  const void *q, *k, *v;  // for the guarded second pass
  int64_t tokens;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  int32_t hq, h, causal;
  int32_t *status;
};

struct Maps {
  CUtensorMap q, k, v;
};

// One softmax warpgroup over its row tile.  Returns false when a wait gave up.
template <typename T>
__device__ __forceinline__ bool softmax_tiles(const Args &a, Smem &S, int t, int tiles, int64_t row, int64_t len,
                                              int64_t row0, uint32_t tmem, float &m_out, float &l_out) {
  constexpr float kSc = kScale * fm::kLog2e;
  const uint32_t lane_base = tmem + (static_cast<uint32_t>((threadIdx.x >> 5) & 3) << 21);  // 32 lanes per warp
  const uint32_t s_at = lane_base + 128 * t, o_at = lane_base + 256 + 128 * t;
  float m = -INFINITY;        // the maximum in use, scaled (log2 units)
  float2 l = make_float2(0.f, 0.f);
  const int64_t seen = a.causal ? min(row + 1, len) : len;  // tokens this row sees
  for (int j = 0; j < tiles; ++j) {
    if (!mbar_wait_bounded(&S.s_full[t], j & 1, a.status)) return false;
    tc::fence_after();
    float s[128];
#pragma unroll
    for (int i = 0; i < 4; ++i) tc::ld32(s + 32 * i, s_at + 32 * i);
    tc::wait_ld();
#pragma unroll
    for (int i = 0; i < 4; ++i) tc::pin32(s + 32 * i);
    const int64_t t0 = static_cast<int64_t>(j) * kN;
    if (a.causal ? t0 + kN > row0 + 1 : t0 + kN > len) {  // some row of the tile does not see all of it
      const int n = static_cast<int>(max(min(seen - t0, int64_t{kN}), int64_t{0}));
#pragma unroll
      for (int i = 0; i < 128; ++i) s[i] = i < n ? s[i] : -INFINITY;
    }
    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int i = 4; i < 128; i += 8) {
#pragma unroll
      for (int c = 0; c < 4; ++c) mx[c] = i + 4 + c < 128 ? fmaxf(mx[c], fmaxf(s[i + c], s[i + 4 + c])) : fmaxf(mx[c], s[i + c]);
    }
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kSc;
    const bool raise = top > m + kRaise;
    if (__any_sync(0xffffffffu, raise)) {
      const float m_new = raise ? top : m;
      if (j > 0) {
        // S of this tile was committed after P.V of the tile before, so O is complete
        const float c = m_new == -INFINITY ? 1.f : fm::ex2(m - m_new);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float o[32];
          tc::ld32(o, o_at + 32 * i);
          tc::wait_ld();
          tc::pin32(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= c;
          tc::st32(o_at + 32 * i, reinterpret_cast<uint32_t *>(o));
        }
        l.x *= c;
        l.y *= c;
      }
      m = m_new;
    }
    const float base = m == -INFINITY ? 0.f : m;
    const float2 sc2 = make_float2(kSc, kSc), nb2 = make_float2(-base, -base);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float2 x = tc::fma2(make_float2(s[32 * i + 2 * e], s[32 * i + 2 * e + 1]), sc2, nb2);
        const float2 y = make_float2(fm::ex2(x.x), fm::ex2(x.y));
        l = tc::add2(l, y);
        p[e] = fm::round_pair<T>(y.x, y.y);
      }
      tc::st16(s_at + 16 * i, p);
    }
    tc::wait_st();
    tc::fence_before();
    tc::mbar_arrive(&S.p_full[t]);
  }
  m_out = m;
  l_out = l.x + l.y;
  return true;
}

// Rows row0 .. row0 + 127 of one head again, with values that a row does not see kept out of
// its products (fm::Rows::tile_guarded): run by a softmax warpgroup (four warps, 16 rows each
// and pass) when its tile had a non-finite output.
template <typename T>
__device__ __noinline__ void redo_rows(const Args &a, uint8_t *smem, int t, int64_t begin, int64_t len,
                                          int64_t row0, int head, int kvh) {
  uint16_t(*ks)[fm::kRow] = reinterpret_cast<uint16_t(*)[fm::kRow]>(smem);
  uint16_t(*vs)[fm::kRow] = ks + fm::kTile;
  const int tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5;
  const T *qb = static_cast<const T *>(a.q) + begin * a.q_tok + head * a.q_head;
  const T *kb = static_cast<const T *>(a.k) + begin * a.k_tok + kvh * a.k_head;
  const T *vb = static_cast<const T *>(a.v) + begin * a.v_tok + kvh * a.v_head;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int64_t first = row0 + 64 * pass, r0 = first + 16 * warp + (lane >> 2), r1 = r0 + 8;
    if (first >= len) break;
    fm::Rows st;
    st.init();
    st.load_q<T>(r0 < len ? qb + r0 * a.q_tok : nullptr, r1 < len ? qb + r1 * a.q_tok : nullptr, lane);
    const int64_t keys = a.causal ? min(len, first + 64) : len;
#pragma unroll 1
    for (int64_t t0 = 0; t0 < keys; t0 += fm::kTile) {
      tc::bar_named(1 + t, 128);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = tid + 128 * i, r = e >> 4, c = (e & 15) * 8;
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (t0 + r < len) {
          x = *reinterpret_cast<const uint4 *>(kb + (t0 + r) * a.k_tok + c);
          y = *reinterpret_cast<const uint4 *>(vb + (t0 + r) * a.v_tok + c);
        }
        *reinterpret_cast<uint4 *>(&ks[r][c]) = x;
        *reinterpret_cast<uint4 *>(&vs[r][c]) = y;
      }
      tc::bar_named(1 + t, 128);
      const int64_t lim0 = (a.causal ? min(len, r0 + 1) : len) - t0, lim1 = (a.causal ? min(len, r1 + 1) : len) - t0;
      st.tile_guarded<T>(ks, vs, static_cast<int>(max(min(lim0, int64_t{64}), int64_t{0})),
                         static_cast<int>(max(min(lim1, int64_t{64}), int64_t{0})), lane);
    }
    float inv[2];
    st.finish(inv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = i ? r1 : r0;
      if (r >= len) continue;
      uint32_t *orow = reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + ((begin + r) * a.hq + head) * kDim);
      int bad = 0;
#pragma unroll
      for (int nt = 0; nt < 16; ++nt) {
        const uint32_t w = fm::round_pair<T>(st.o[nt][2 * i] * inv[i], st.o[nt][2 * i + 1] * inv[i]);
        orow[4 * nt + (lane & 3)] = w;
        const float2 x = Elem<T>::to_f2(w);
        bad |= !isfinite(x.x) || !isfinite(x.y);
      }
      if (bad) set_status(a.status, NSNKV_ST_OUTPUT_NONFINITE);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) prompt_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps) {
  extern __shared__ uint8_t smem_raw[];
  // the swizzle's pattern repeats every 1024 bytes of the shared address
  Smem &S = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  const int tid = threadIdx.x, warp = tid >> 5;
  const int head = blockIdx.x, kvh = head / (a.hq / a.h);
  const int64_t begin = min(max(static_cast<int64_t>(a.cu[blockIdx.y]), int64_t{0}), a.tokens);
  const int64_t len = min(max(static_cast<int64_t>(a.cu[blockIdx.y + 1]), begin), a.tokens) - begin;
  // longest row tiles first: block z counts them down
  const int64_t pair = static_cast<int64_t>(gridDim.z) - 1 - blockIdx.z;
  const int64_t row0 = pair * 2 * kM;
  if (row0 >= len) return;
  int tiles[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int64_t first = row0 + t * kM;
    const int64_t keys = a.causal ? min(first + kM, len) : len;
    tiles[t] = first < len ? static_cast<int>((keys + kN - 1) / kN) : 0;
  }
  const int all = max(tiles[0], tiles[1]);

  if (warp == 8) {
    tc::tmem_alloc(&S.tmem, 512);
  } else if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.q_full[i], 1);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i], 128);
      mbar_init(&S.o_full[i], 1);
      S.redo[i] = 0;
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&S.kv_full[i], 1);
      mbar_init(&S.kv_empty[i], 1);
    }
    S.failed = 0;
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = S.tmem;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9 && tc::elect()) {  // ---- TMA loads; ring tile 2 j is K_j, 2 j + 1 is V_j
      tc::prefetch_map(&maps.q);
      tc::prefetch_map(&maps.k);
      tc::prefetch_map(&maps.v);
      auto load = [&](uint8_t *dst, const CUtensorMap &map, int hd, int64_t tok, uint64_t *bar) {
        mbar_expect_tx(bar, kTileBytes);
        tc::tma_load_3d(dst, &map, 0, hd, static_cast<int>(tok), bar);
        tc::tma_load_3d(dst + kTileBytes / 2, &map, 64, hd, static_cast<int>(tok), bar);
      };
      auto ring = [&](int i) {
        load(S.kv[i % kStages], i & 1 ? maps.v : maps.k, kvh, begin + static_cast<int64_t>(i >> 1) * kN,
             &S.kv_full[i % kStages]);
      };
      load(S.q[0], maps.q, head, begin + row0, &S.q_full[0]);
      ring(0);
      if (tiles[1] > 0) load(S.q[1], maps.q, head, begin + row0 + kM, &S.q_full[1]);
      int i = 1;
      bool ok = true;
      for (; i < 2 * all && ok; ++i) {
        if (i >= kStages) ok = mbar_wait_bounded(&S.kv_empty[i % kStages], (i / kStages - 1) & 1, a.status);
        if (ok) ring(i);
      }
      if (!ok) {  // give up, but not before the copies in flight have landed
        --i;
        for (int x = max(0, i - kStages); x < i; ++x)
          mbar_wait_bounded(&S.kv_full[x % kStages], (x / kStages) & 1, a.status);
      }
    } else if (warp == 8 && tc::elect()) {  // ---- MMA
      constexpr uint32_t kIdS = tc::instr_desc<T>(kM, kN, false), kIdO = tc::instr_desc<T>(kM, kDim, true);
      auto scores = [&](int t, int slot) {
        const uint32_t qa = tc::saddr(S.q[t]), ka = tc::saddr(S.kv[slot]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = (k >> 2) * (kTileBytes / 2) + (k & 3) * 32;
          tc::mma_ss(tmem + 128 * t, tc::smem_desc(qa + off, 16, 1024), tc::smem_desc(ka + off, 16, 1024), kIdS, k > 0);
        }
        tc::commit(&S.s_full[t]);
      };
      auto values = [&](int t, int slot, bool acc) {
        const uint32_t va = tc::saddr(S.kv[slot]);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          tc::mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k,
                     tc::smem_desc(va + k * 2048, kTileBytes / 2, 1024), kIdO, acc || k > 0);
        tc::commit(&S.o_full[t]);
      };
      auto ready = [&](int i) { return mbar_wait_bounded(&S.kv_full[i % kStages], (i / kStages) & 1, a.status); };
      bool ok = ready(0);
      for (int t = 0; t < 2 && ok; ++t) {
        if (tiles[t] == 0) continue;
        ok = mbar_wait_bounded(&S.q_full[t], 0, a.status);
        tc::fence_after();
        if (ok) scores(t, 0);
      }
      tc::commit(&S.kv_empty[0]);
      for (int j = 0; j < all && ok; ++j) {
        const int vi = 2 * j + 1, ki = 2 * j + 2;
        ok = ready(vi);
        bool have_k = false;
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= tiles[t]) continue;
          ok = mbar_wait_bounded(&S.p_full[t], j & 1, a.status);
          if (!ok) break;
          tc::fence_after();
          values(t, vi % kStages, j > 0);
          if (j + 1 < tiles[t]) {
            if (!have_k) {
              ok = ready(ki);
              have_k = true;
              if (!ok) break;
            }
            scores(t, ki % kStages);
          }
        }
        tc::commit(&S.kv_empty[vi % kStages]);
        if (have_k) tc::commit(&S.kv_empty[ki % kStages]);
      }
      if (!ok) S.failed = 1;
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2;
    const int64_t first = row0 + t * kM, row = first + (tid & 127);
    if (tiles[t] > 0) {
      float m, l;
      bool ok = softmax_tiles<T>(a, S, t, tiles[t], row, len, first, tmem, m, l);
      ok = ok && mbar_wait_bounded(&S.o_full[t], (tiles[t] - 1) & 1, a.status);
      if (ok) {
        tc::fence_after();
        const float inv = m == -INFINITY ? 0.f : __fdiv_rn(1.f, l);
        const uint32_t o_at = tmem + (static_cast<uint32_t>(warp & 3) << 21) + 256 + 128 * t;
        T *orow = static_cast<T *>(a.out) + ((begin + row) * a.hq + head) * kDim;
        int bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float o[32];
          tc::ld32(o, o_at + 32 * i);
          tc::wait_ld();
          tc::pin32(o);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            w[e] = fm::round_pair<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
            const float2 x = Elem<T>::to_f2(w[e]);
            bad |= !isfinite(x.x) || !isfinite(x.y);
          }
          if (row < len)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              reinterpret_cast<uint4 *>(orow)[4 * i + e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        }
        if (bad && row < len) S.redo[t] = 1;
        if (a.lse && row < len)
          a.lse[(begin + row) * a.hq + head] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * fm::kLn2;
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::tmem_release(tmem, 512);
  // Every copy and MMA has finished: the K / V ring is free for the guarded pass.
  if (warp < 8 && S.redo[warp >> 2] && !S.failed)
    redo_rows<T>(a, S.kv[2 * (warp >> 2)], warp >> 2, begin, len, row0 + (warp >> 2) * kM, head, kvh);
}

}  // namespace ptc
}  // namespace nsnkv
