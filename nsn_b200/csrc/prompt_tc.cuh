// Prompt attention on the tensor cores (tcgen05), for prompts of a few tiles and more.
//
// One CTA per SM takes items of 256 query rows of one head (two 128-row tiles) and attends
// them over 128-token K / V tiles:
//   warps 0-3, 4-7   softmax of row tile 0 and 1, one row per thread
//   warp 8           issues the MMAs, one thread
//   warp 9           issues the TMA loads: Q per item, K and V through a ring of kStages tiles
//   warp 10          lays out the items ahead of the others
// The code that runs once per item or rarely is kept small (rolled loops, calls): the four
// schedulers of an SM fetch the softmax loop and the issue loops side by side, and what does
// not fit their instruction caches stalls every warp.
// TMEM (512 columns): S0 | S1 | O0 | O1.  Per tile and row tile: S = Q.K^T into S; the
// softmax warps read a row of S into registers, write P = 2^(x - m) in 16 bits over S and the
// tensor core adds P.V to O, P read from TMEM.  While one row tile is in its softmax the
// tensor core works on the other.
//
// Measured: 16384 tokens, GQA 32:8, fp16: 1.76 ms in a short run (1250 TFLOP/s, 0.76 of the
// library GEMM's burst rate), 2.12 ms under sustained load, where the power limit holds the clock;
// 4 x 2048 tokens, 16 heads: 99 us.  What bounds it is the chain S -> softmax -> P.V of one row
// tile with one warp per scheduler (about 2450 of 3150 cycles per K / V tile are softmax); the
// tensor pipe is busy 43% to 50% of the time.  Tiles are 128 tokens because Q.K^T with both operands in shared
// memory reads 128 bytes a cycle at N = 128, all that shared memory gives, and more below.
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

constexpr int kItems = 4;  // items laid out ahead

struct Smem {
  uint8_t q[2][kTileBytes];        // each [2 halves of 64 channels][128 rows][128 B swizzled]
  uint8_t kv[kStages][kTileBytes];
  uint64_t q_full[2], q_empty[2], kv_full[kStages], kv_empty[kStages], s_full[2], p_full[2][2], o_full[2];
  uint64_t item_full[kItems], item_empty[kItems];
  int32_t item[kItems][8];
  uint32_t tmem;
  int32_t failed;
  uint32_t redo[2][32];
};

struct Args {
  const int32_t *cu;
  void *out;
  float *lse;
  const void *q, *k, *v;  // for the guarded second pass
  int64_t tokens;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  int32_t seqs, hq, h, causal;
  int32_t *status;
};

struct Maps {
  CUtensorMap q, k, v;
};

// One softmax warpgroup over its row tile.  P is announced in two halves of 64 tokens: the P.V
// MMAs of the first run while the second is computed.
template <typename T>
__device__ __forceinline__ void softmax_tiles(const Args &a, Smem &S, int t, int tiles, uint32_t done, int row, int len,
                                              int row0, uint32_t tmem, float &m_out, float &l_out) {
  constexpr float kSc = kScale * fm::kLog2e;
  const uint32_t lane_base = tmem + (static_cast<uint32_t>((threadIdx.x >> 5) & 3) << 21);  // 32 lanes per warp
  const uint32_t s_at = lane_base + 128 * t, o_at = lane_base + 256 + 128 * t;
  float m = -INFINITY;        // the maximum in use, scaled (log2 units)
  float2 l = make_float2(0.f, 0.f), l2 = l;
  const int seen = a.causal ? min(row + 1, len) : len;  // tokens this row sees
  const int whole = a.causal ? row0 + 1 : len;          // tokens every row of the tile sees
  for (int j = 0; j < tiles; ++j) {
    tc::wait(&S.s_full[t], (done + j) & 1, &S.failed, a.status);
    tc::fence_after();
    // Two rolled passes over halves of 64 tokens (maximum; exponentials), S read from TMEM in
    // each: half the code of an unrolled tile.
    float s[64], mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    const int n = seen - j * kN;
    const bool masked = j * kN + kN > whole;  // some row of the tile does not see all of it
    auto load = [&](int h) {
      tc::ld32(s, s_at + 64 * h);
      tc::ld32(s + 32, s_at + 64 * h + 32);
      tc::wait_ld();
      tc::pin32(s);
      tc::pin32(s + 32);
      if (masked) {
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] = i < n - 64 * h ? s[i] : -INFINITY;
      }
    };
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      load(h);
#pragma unroll
      for (int i = 0; i < 64; i += 8)
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = tc::max3(mx[c], s[i + c], s[i + 4 + c]);
    }
    const float top = kSc * fmaxf(tc::max3(mx[0], mx[1], mx[2]), mx[3]);
    const bool raise = top > m + kRaise;
    if (__any_sync(0xffffffffu, raise)) {
      const float m_new = raise ? top : m;
      if (j > 0) {
        // S of this tile was committed after P.V of the tile before, so O is complete
        const float c = m_new == -INFINITY ? 1.f : fm::ex2(m - m_new);
#pragma unroll 1
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
        l2.x *= c;
        l2.y *= c;
      }
      m = m_new;
    }
    const float base = m == -INFINITY ? 0.f : m;
    const float2 sc2 = make_float2(kSc, kSc), nb2 = make_float2(-base, -base);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      load(h);
      uint32_t p[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float2 x = tc::fma2(make_float2(s[2 * e], s[2 * e + 1]), sc2, nb2);
        const float2 y = make_float2(fm::ex2(x.x), fm::ex2(x.y));
        if (e & 1) l2 = tc::add2(l2, y); else l = tc::add2(l, y);
        p[e] = fm::round_pair<T>(y.x, y.y);
      }
      tc::st32(s_at + 32 * h, p);
      tc::wait_st();
      tc::fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&S.p_full[t][h]);
    }
  }
  l = tc::add2(l, l2);
  m_out = m;
  l_out = l.x + l.y;
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

// A position in the K / V ring: stage and the parity of its barriers.
struct Ring {
  uint32_t slot, phase;
  __device__ __forceinline__ void next() {
    if (++slot == kStages) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Work items: (row-tile pair of a sequence, head), longest first: pair p of every sequence that
// has one before pair p - 1, heads innermost, so that the CTAs running together share K and V
// in L2 and the short items come last.  Warp-collective: lane i holds the pair counts of
// sequences i, i + 32, ...  Batches of more than 128 sequences keep the sequences' order.
struct Item {
  int begin, len, row0, head;  // the sequence's first token and length, the pair's first row
  int tiles[2];                // K / V tiles of each row tile; tiles[0] = 0 ends the list
  int pad[2];
};

struct Schedule {
  int np[4];
  uint32_t pairs;

  __device__ __forceinline__ void range(const Args &a, int s, int64_t &begin, int64_t &len) const {
    begin = min(max(static_cast<int64_t>(a.cu[s]), int64_t{0}), a.tokens);
    len = min(max(static_cast<int64_t>(a.cu[s + 1]), begin), a.tokens) - begin;
  }
  __device__ __forceinline__ int count(const Args &a, int s) const {
    if (s >= a.seqs) return 0;
    int64_t begin, len;
    range(a, s, begin, len);
    return static_cast<int>((len + 2 * kM - 1) / (2 * kM));
  }
  __device__ __forceinline__ void init(const Args &a) {
    const int lane = threadIdx.x & 31;
    pairs = 0;
    if (a.seqs <= 128) {
      int n = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        np[c] = count(a, lane + 32 * c);
        n += np[c];
      }
      pairs = __reduce_add_sync(0xffffffffu, n);
    } else {
      for (int s = 0; s < a.seqs; s += 32) pairs += __reduce_add_sync(0xffffffffu, count(a, s + lane));
    }
  }
  // pairs at level p or above, over all sequences
  __device__ __forceinline__ int above(int p) const {
    int n = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) n += max(np[c] - p, 0);
    return __reduce_add_sync(0xffffffffu, n);
  }
  __device__ __forceinline__ bool item(const Args &a, uint32_t k, Item &it) const {
    const uint32_t g = gridDim.x, c = blockIdx.x, hq = a.hq;
    const uint32_t rank = static_cast<uint32_t>(k) * g + (k & 1 ? g - 1 - c : c);  // back and forth over the CTAs
    it.tiles[0] = it.tiles[1] = 0;
    if (rank >= pairs * hq) return false;
    const int lane = threadIdx.x & 31;
    it.head = static_cast<int>(rank % hq);
    int r = static_cast<int>(rank / hq), seq = 0, pair = 0;
    if (a.seqs <= 128) {
      int lo = 0, hi = __reduce_max_sync(0xffffffffu, max(max(np[0], np[1]), max(np[2], np[3])));
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (above(mid) > r) lo = mid; else hi = mid;
      }
      r -= above(lo + 1);
      pair = lo;
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const uint32_t has = __ballot_sync(0xffffffffu, np[c4] > lo);
        const uint32_t mine = __ballot_sync(0xffffffffu, np[c4] > lo && __popc(has & ((1u << lane) - 1u)) == r);
        if (mine) seq = 32 * c4 + __ffs(mine) - 1;
        r -= __popc(has);
      }
    } else {
      for (int s = 0; s < a.seqs; s += 32) {
        const int n = count(a, s + lane);
        int up = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, up, d);
          if (lane >= d) up += x;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, up > r);
        if (past) {
          const int at = __ffs(past) - 1;
          seq = s + at;
          pair = __shfl_sync(0xffffffffu, n - up, at) + r;
          break;
        }
        r -= __shfl_sync(0xffffffffu, up, 31);
      }
    }
    int64_t begin, len;
    range(a, seq, begin, len);
    it.begin = static_cast<int>(begin);
    it.len = static_cast<int>(len);
    it.row0 = pair * 2 * kM;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int first = it.row0 + t * kM;
      const int keys = a.causal ? min(first + kM, it.len) : it.len;
      it.tiles[t] = first < it.len ? (keys + kN - 1) / kN : 0;
    }
    return true;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ Maps maps) {
  extern __shared__ uint8_t smem_raw[];
  // the swizzle's pattern repeats every 1024 bytes of the shared address
  Smem &S = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  const int tid = threadIdx.x, warp = tid >> 5;
  const int group = a.hq / a.h;

  if (warp == 8) {
    tc::tmem_alloc(&S.tmem, 512);
  } else if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.q_full[i], 1);
      mbar_init(&S.q_empty[i], 1);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i][0], 4);  // one arrival per softmax warp
      mbar_init(&S.p_full[i][1], 4);
      mbar_init(&S.o_full[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&S.kv_full[i], 1);
      mbar_init(&S.kv_empty[i], 1);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&S.item_full[i], 1);
      mbar_init(&S.item_empty[i], 10);  // the loader, the MMA warp and eight softmax warps
    }
    S.failed = 0;
    fence_mbar_init();
  }
  if (warp == 1) S.redo[0][tid & 31] = S.redo[1][tid & 31] = 0;
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = S.tmem;
  // Item k of this CTA, read by a whole warp; false at the end of the list.
  auto item = [&](uint32_t k, Item &it) {
    const uint32_t slot = k % kItems;
    tc::wait(&S.item_full[slot], k / kItems & 1, &S.failed, a.status);
    const int4 x = reinterpret_cast<const int4 *>(S.item[slot])[0], y = reinterpret_cast<const int4 *>(S.item[slot])[1];
    it.begin = x.x, it.len = x.y, it.row0 = x.z, it.head = x.w;
    // the broadcast tells the compiler that the loop bounds are the warp's
    it.tiles[0] = __shfl_sync(0xffffffffu, y.x, 0), it.tiles[1] = __shfl_sync(0xffffffffu, y.y, 0);
    if ((tid & 31) == 0) tc::mbar_arrive(&S.item_empty[slot]);
    return it.tiles[0] > 0 && !*static_cast<volatile int32_t *>(&S.failed);
  };

  if (warp >= 8) {
    if (warp == 10) {  // ---- items
      Schedule sch;
      sch.init(a);
      Item it;
      bool more = true;
      for (uint32_t k = 0; more; ++k) {
        more = sch.item(a, k, it);
        tc::wait(&S.item_empty[k % kItems], (k / kItems & 1) ^ 1, &S.failed, a.status);
        if (*static_cast<volatile int32_t *>(&S.failed)) it.tiles[0] = 0, more = false;
        if ((tid & 31) == 0) {
          reinterpret_cast<int4 *>(S.item[k % kItems])[0] = make_int4(it.begin, it.len, it.row0, it.head);
          reinterpret_cast<int4 *>(S.item[k % kItems])[1] = make_int4(it.tiles[0], it.tiles[1], 0, 0);
          tc::mbar_arrive(&S.item_full[k % kItems]);
        }
        __syncwarp();
      }
    } else if (warp == 9) {  // ---- TMA loads; ring tile 2 j is K_j, 2 j + 1 is V_j
      const bool lead = tc::elect();
      if (lead) {
        tc::prefetch_map(&maps.q);
        tc::prefetch_map(&maps.k);
        tc::prefetch_map(&maps.v);
      }
      auto load = [&](uint8_t *dst, const CUtensorMap *map, int hd, int tok, uint64_t *bar) {
        mbar_expect_tx(bar, kTileBytes);
        tc::tma_load_3d(dst, map, 0, hd, tok, bar);
        tc::tma_load_3d(dst + kTileBytes / 2, map, 64, hd, tok, bar);
      };
      Ring at{0, 1};    // a fresh barrier counts as the phase before: the first round does not wait
      uint32_t qn = 0;  // bit t: parity of Q loads of row tile t
      Item it;
      for (uint32_t k = 0; item(k, it); ++k) {
        const int kvh = it.head / group, all = max(it.tiles[0], it.tiles[1]);
        // Q of row tile 0, K_0, Q of row tile 1, V_0, K_1, ...
        auto queries = [&](int t) {
          if (it.tiles[t] == 0) return;
          tc::wait(&S.q_empty[t], (qn >> t & 1) ^ 1, &S.failed, a.status);
          qn ^= 1u << t;
          if (lead) load(S.q[t], &maps.q, it.head, it.begin + it.row0 + t * kM, &S.q_full[t]);
        };
        queries(0);
#pragma unroll 1
        for (int i = 0; i < 2 * all; ++i) {
          tc::wait(&S.kv_empty[at.slot], at.phase, &S.failed, a.status);
          if (lead) load(S.kv[at.slot], i & 1 ? &maps.v : &maps.k, kvh, it.begin + (i >> 1) * kN, &S.kv_full[at.slot]);
          at.next();
          if (i == 0) queries(1);
        }
      }
      if (*static_cast<volatile int32_t *>(&S.failed))  // a wait gave up: let the copies in flight land
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 8) {  // ---- MMA
      // Every lane runs the loops and the waits, so that addresses and descriptors stay in uniform
      // registers; one lane issues.
      const bool lead = tc::elect();
      constexpr uint32_t kIdS = tc::instr_desc<T>(kM, kN, false), kIdO = tc::instr_desc<T>(kM, kDim, true);
      // descriptors in 16-byte units: adding to them moves the start address
      const uint64_t qd = tc::smem_desc(tc::saddr(S.q[0]), 16, 1024), kd = tc::smem_desc(tc::saddr(S.kv[0]), 16, 1024),
                     vd = tc::smem_desc(tc::saddr(S.kv[0]), kTileBytes / 2, 1024);
      auto scores = [&](int t, uint32_t slot) {
        const uint64_t qa = qd + t * (kTileBytes >> 4), ka = kd + slot * (kTileBytes >> 4);
        tc::fence_after();
        if (lead) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t off = ((i >> 2) * (kTileBytes / 2) + (i & 3) * 32) >> 4;
            tc::mma_ss(tmem + 128 * t, qa + off, ka + off, kIdS, i > 0);
          }
          tc::commit(&S.s_full[t]);
        }
      };
      auto values = [&](int t, int h, uint32_t slot, bool acc) {
        const uint64_t va = vd + slot * (kTileBytes >> 4) + h * (4 * 2048 >> 4);
        tc::fence_after();
        if (lead) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            tc::mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 32 * h + 8 * i, va + i * (2048 >> 4), kIdO, acc || i > 0);
        }
      };
      auto signal = [&](uint64_t *bar) {
        if (lead) tc::commit(bar);
      };
      auto ready = [&](const Ring &r) { tc::wait(&S.kv_full[r.slot], r.phase, &S.failed, a.status); };
      Ring at{0, 0};            // the ring position of the next K or V tile
      uint32_t qn = 0, pn = 0;  // bit t: parity of the next Q tile, P tile of row tile t
      auto first = [&](int t, int tiles, const Ring &r) {  // S of an item's first tile
        tc::wait(&S.q_full[t], qn >> t & 1, &S.failed, a.status);
        qn ^= 1u << t;
        ready(r);
        scores(t, r.slot);
        if (tiles == 1) signal(&S.q_empty[t]);
      };
      Item it, next;
      bool more = item(0, it), ahead = false;
      for (uint32_t k = 0; more; ++k) {
        more = item(k + 1, next);
        const int n0 = it.tiles[0], n1 = it.tiles[1], all = max(n0, n1);
        if (!ahead) first(0, n0, at);  // row tile 0 of an item is never empty
        ahead = false;
        if (n1 > 0) first(1, n1, at);
        signal(&S.kv_empty[at.slot]);
        at.next();
#pragma unroll 1
        for (int j = 0; j < all; ++j) {  // P.V of tile j, S of tile j + 1
          Ring kr = at;                  // V_j at `at`, K_{j + 1} (or the next item's K_0) behind it
          kr.next();
          ready(at);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int n = t ? n1 : n0;
            if (j < n) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                tc::wait(&S.p_full[t][h], pn >> t & 1, &S.failed, a.status);
                values(t, h, at.slot, j > 0 || h > 0);
              }
              pn ^= 1u << t;
              if (j + 1 < n) {
                ready(kr);
                scores(t, kr.slot);
                if (j + 2 == n) signal(&S.q_empty[t]);
              } else {
                signal(&S.o_full[t]);
              }
            } else if (t == 0 && more) {
              // row tile 0 is done: start it on the next item while row tile 1 finishes
              first(0, next.tiles[0], kr);
              ahead = true;
            }
          }
          signal(&S.kv_empty[at.slot]);
          if (j + 1 < all) {
            signal(&S.kv_empty[kr.slot]);
            kr.next();
          }
          at = kr;
        }
        it = next;
      }
    }
    __syncwarp();
  } else {
    const int t = warp >> 2;
    uint32_t done = 0, taken = 0;  // S tiles and finished O tiles taken so far
    Item it;
    for (uint32_t k = 0; item(k, it); ++k) {
      const int tiles = it.tiles[t];
      if (tiles == 0) continue;
      const int first = it.row0 + t * kM, row = first + (tid & 127);
      float m, l;
      softmax_tiles<T>(a, S, t, tiles, done, row, it.len, first, tmem, m, l);
      done += tiles;
      tc::wait(&S.o_full[t], taken & 1, &S.failed, a.status);
      ++taken;
      tc::fence_after();
      const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);  // l: 0 if the row saw nothing, NaN if only NaN
      const uint32_t o_at = tmem + (static_cast<uint32_t>(warp & 3) << 21) + 256 + 128 * t;
      const int64_t at = static_cast<int64_t>(it.begin + row) * a.hq + it.head;
      T *orow = static_cast<T *>(a.out) + at * kDim;
      uint32_t check = 0;  // 0 * w summed: NaN when a rounded output is not finite
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        float o[32];
        tc::ld32(o, o_at + 32 * i);
        tc::wait_ld();
        tc::pin32(o);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 y = tc::mul2(make_float2(o[2 * e], o[2 * e + 1]), make_float2(inv, inv));
          w[e] = fm::round_pair<T>(y.x, y.y);
          check = fm::add_zero_times<T>(check, w[e]);
        }
        if (row < it.len) {
          tc::store32(orow + 32 * i, w);
          tc::store32(orow + 32 * i + 16, w + 8);
        }
      }
      tc::fence_before();  // O is read before the next item's first P is announced
      if (row < it.len) {
        const float2 nan = Elem<T>::to_f2(check);
        if (nan.x + nan.y != 0.f) atomicOr(&S.redo[t][k >> 5 & 31], 1u << (k & 31));
        if (a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * fm::kLn2;
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::tmem_release(tmem, 512);
  // Items with a non-finite output once more, guarded; every copy and MMA has finished, so the
  // ring is free.  (Item k of the CTA is bit k mod 1024: one more item than needed may run.)
  if (warp < 8 && !S.failed) {
    const int t = warp >> 2;
    if (__any_sync(0xffffffffu, S.redo[t][tid & 31] != 0)) {
      Schedule sch;
      sch.init(a);
      Item it;
      for (uint32_t k = 0; sch.item(a, k, it); ++k)
        if (S.redo[t][k >> 5 & 31] >> (k & 31) & 1 && it.tiles[t] > 0)
          redo_rows<T>(a, S.kv[2 * t], t, it.begin, it.len, it.row0 + t * kM, it.head, it.head / group);
    }
  }
}

}  // namespace ptc
}  // namespace nsnkv
