// Attention over a sealed prefix that many query rows share (include/nsnkv.h,
// nsnkv_prefix_attn): the prefix's block records are read and restored once per kv head for
// all rows of a group, instead of once per sequence.
//
// A group's rows are (query row, query head) pairs: position p = r / G of the group and head
// g = r % G of the kv head's G = hq / h.  The prefix is split into chunks of pages; every
// (chunk, kv head, row tile) writes its rows' normalised output and log-sum-exp, and one
// merge joins the chunks and the row's attention over its own tokens (o_part, lse_part):
//   out = sum_i 2^(e_i - E) o_i,  E = log2 sum_i 2^e_i.
#include "flash_mma.cuh"
#include "record_rows.cuh"

namespace nsnkv {
namespace {

struct PrefixArgs {
  const void *q;
  const uint8_t *records;
  const int32_t *table, *n_pages, *row_offsets, *row_index;
  const float *o_part, *lse_part;
  void *out;
  float *lse;
  float *o_ws, *e_ws;  // [chunks][rows][hq][128], [chunks][rows][hq] (base-2 log-sum-exp)
  int64_t rows, pages, table_stride, rec_head, rec_page;  // record strides in bytes
  int32_t groups, hq, h, max_pages, chunk_pages, row_tiles;
  int32_t *status;
};

__device__ __forceinline__ int group_pages(const PrefixArgs &a, int g) {
  return min(max(a.n_pages ? a.n_pages[g] : a.max_pages, 0), a.max_pages);
}
// Positions [begin, end) of group g in the row order.
__device__ __forceinline__ void group_rows(const PrefixArgs &a, int g, int64_t &begin, int64_t &end) {
  begin = a.row_offsets ? min(max(static_cast<int64_t>(a.row_offsets[g]), int64_t{0}), a.rows) : 0;
  end = a.row_offsets ? min(max(static_cast<int64_t>(a.row_offsets[g + 1]), begin), a.rows) : a.rows;
}
// The query row at position p; -1 when the index names no row.
__device__ __forceinline__ int64_t row_at(const PrefixArgs &a, int64_t p) {
  if (!a.row_index) return p;
  const int64_t r = a.row_index[p];
  return r >= 0 && r < a.rows ? r : -1;
}

constexpr int kRowsCta = 64;

template <int BITS>
struct PrefixSmem {
  uint8_t rec[2][rr::Rec<BITS>::kBytes];
  uint16_t k[fm::kTile][fm::kRow];
  uint16_t v[fm::kTile][fm::kRow];
  uint64_t full[2];
};

// One block's K and V rows into the tiles, 128 threads.
template <int BITS, typename T>
__device__ __forceinline__ int restore_block(const uint8_t *rec, uint16_t (*ks)[fm::kRow], uint16_t (*vs)[fm::kRow],
                                             int tid) {
  using R = rr::Rec<BITS>;
  int bad = 0;
  uint32_t a[16], b[16], w[BITS];
  {
    const int g = tid & 3;
    __half2 mn[16], sc[16];
    const __half2 *pm = reinterpret_cast<const __half2 *>(rec + R::kMin) + 16 * g;
    const __half2 *ps = reinterpret_cast<const __half2 *>(rec + R::kScaleAt) + 16 * g;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      mn[i] = pm[i];
      sc[i] = ps[i];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = (tid >> 2) + 32 * e;
      const float alpha = reinterpret_cast<const float *>(rec + R::kAlpha)[t];
#pragma unroll
      for (int i = 0; i < BITS; ++i) w[i] = reinterpret_cast<const uint32_t *>(rec)[t * 4 * BITS + g * BITS + i];
      rr::codes16<BITS>(w, a, b);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        *reinterpret_cast<uint4 *>(&ks[t][32 * g + 8 * c]) = rr::values8<T>(a + 8 * c, mn + 4 * c, sc + 4 * c, alpha);
        *reinterpret_cast<uint4 *>(&ks[t][32 * g + 16 + 8 * c]) =
            rr::values8<T>(b + 8 * c, mn + 8 + 4 * c, sc + 8 + 4 * c, alpha);
      }
      bad |= !isfinite(alpha);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 m = __half22float2(mn[i]), s = __half22float2(sc[i]);
      bad |= !isfinite(m.x) || !isfinite(m.y) || !isfinite(s.x) || !isfinite(s.y);
    }
  }
  {
    const uint8_t *vr = rec + R::kHalf;
    const int c16 = tid & 7;
    __half2 mn[8], sc[8];
    const __half2 *pm = reinterpret_cast<const __half2 *>(vr + R::kMin) + 8 * c16;
    const __half2 *ps = reinterpret_cast<const __half2 *>(vr + R::kScaleAt) + 8 * c16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mn[i] = pm[i];
      sc[i] = ps[i];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = (tid >> 3) + 16 * e;
      const float2 alpha = reinterpret_cast<const float2 *>(vr + R::kAlpha)[j];
#pragma unroll
      for (int i = 0; i < BITS; ++i) w[i] = reinterpret_cast<const uint32_t *>(vr)[j * 8 * BITS + c16 * BITS + i];
      rr::codes16<BITS>(w, a, b);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        *reinterpret_cast<uint4 *>(&vs[2 * j][16 * c16 + 8 * c]) =
            rr::values8<T>(a + 8 * c, mn + 4 * c, sc + 4 * c, alpha.x);
        *reinterpret_cast<uint4 *>(&vs[2 * j + 1][16 * c16 + 8 * c]) =
            rr::values8<T>(b + 8 * c, mn + 4 * c, sc + 4 * c, alpha.y);
      }
      bad |= !isfinite(alpha.x) || !isfinite(alpha.y);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 m = __half22float2(mn[i]), s = __half22float2(sc[i]);
      bad |= !isfinite(m.x) || !isfinite(m.y) || !isfinite(s.x) || !isfinite(s.y);
    }
  }
  return bad;
}

// One chunk of pages, one kv head, 64 rows at a time (16 per warp).
template <int BITS, typename T>
__global__ void __launch_bounds__(128, 3) prefix_rows_kernel(const PrefixArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  PrefixSmem<BITS> &S = *reinterpret_cast<PrefixSmem<BITS> *>(smem_raw);
  constexpr uint32_t kBytes = rr::Rec<BITS>::kBytes;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = blockIdx.x, head = blockIdx.y;
  const int group = blockIdx.z / a.row_tiles, G = a.hq / a.h;
  const int np = group_pages(a, group), p0 = chunk * a.chunk_pages;
  if (p0 >= np) return;
  const int nloc = min(a.chunk_pages, np - p0);
  int64_t begin, end;
  group_rows(a, group, begin, end);
  const int64_t nrows = (end - begin) * G;
  if (tid == 0) {
    mbar_init(&S.full[0], 1);
    mbar_init(&S.full[1], 1);
    fence_mbar_init();
  }
  __syncthreads();
  const int32_t *row = a.table + group * a.table_stride + p0;
  uint32_t phase[2] = {0u, 0u};
  int bad = 0;
  for (int64_t rt = blockIdx.z % a.row_tiles; rt * kRowsCta < nrows; rt += a.row_tiles) {
    auto issue = [&](int i) {  // thread 0: record i of the chunk into slot i & 1
      int64_t page = row[i];
      if (page < 0 || page >= a.pages) {
        set_status(a.status, NSNKV_ST_PAGE);
        page = 0;
      }
      mbar_expect_tx(&S.full[i & 1], kBytes);
      bulk_g2s(S.rec[i & 1], a.records + head * a.rec_head + page * a.rec_page, kBytes, &S.full[i & 1]);
    };
    if (tid == 0) issue(0);
    int64_t out_at[2];
    const T *qp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = rt * kRowsCta + 16 * warp + (lane >> 2) + 8 * i;
      const int64_t qr = r < nrows ? row_at(a, begin + r / G) : -1;
      const int64_t at = qr * a.hq + head * G + r % G;
      out_at[i] = qr < 0 ? -1 : at;
      qp[i] = qr < 0 ? nullptr : static_cast<const T *>(a.q) + at * kDim;
    }
    fm::Rows st;
    st.init();
    st.load_q<T>(qp[0], qp[1], lane);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = Elem<T>::to_f2(st.q[ks][i]);
        bad |= !isfinite(x.x) || !isfinite(x.y);
      }
    const bool active = rt * kRowsCta + 16 * warp < nrows;  // this warp has rows
    for (int i = 0; i < nloc; ++i) {
      if (!__syncthreads_and(mbar_wait_bounded(&S.full[i & 1], phase[i & 1], a.status))) return;
      phase[i & 1] ^= 1u;
      if (tid == 0 && i + 1 < nloc) issue(i + 1);  // its slot was read before the last barrier
      bad |= restore_block<BITS, T>(S.rec[i & 1], S.k, S.v, tid);
      __syncthreads();
      if (active) st.tile<T>(S.k, S.v, fm::kTile, fm::kTile, lane);
      __syncthreads();
    }
    float inv[2];
    st.finish(inv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (out_at[i] < 0) continue;
      const int64_t at = chunk * a.rows * a.hq + out_at[i];
#pragma unroll
      for (int nt = 0; nt < 16; ++nt)
        reinterpret_cast<float2 *>(a.o_ws + at * kDim)[4 * nt + (lane & 3)] =
            make_float2(st.o[nt][2 * i] * inv[i], st.o[nt][2 * i + 1] * inv[i]);
      if ((lane & 3) == 0) a.e_ws[at] = st.lse2(i);
    }
  }
  if (bad) set_status(a.status, NSNKV_ST_INPUT_NONFINITE);
}

// One warp per (query row, head): the chunks of its group and its own partial.
template <typename T>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (item >= a.rows * a.hq) return;
  const int64_t p = item / a.hq, head = item % a.hq;
  const int64_t r = row_at(a, p);
  if (r < 0) return;
  int chunks = 0;
  for (int g = 0; g < a.groups; ++g) {
    int64_t begin, end;
    group_rows(a, g, begin, end);
    if (p >= begin && p < end) chunks = (group_pages(a, g) + a.chunk_pages - 1) / a.chunk_pages;
  }
  const int64_t at = r * a.hq + head, step = a.rows * a.hq;
  float m = a.lse_part ? a.lse_part[at] * fm::kLog2e : -INFINITY;
  const float own = m;
  for (int c = 0; c < chunks; ++c) m = fmaxf(m, a.e_ws[c * step + at]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float e, const float *row) {
    const float w = fm::ex2(e - base);
    if (e == -INFINITY) return;  // nothing seen: its row is not read
    const float4 x = reinterpret_cast<const float4 *>(row)[lane];
    l += w;
    o.x += w * x.x;
    o.y += w * x.y;
    o.z += w * x.z;
    o.w += w * x.w;
  };
  if (a.o_part) add(own, a.o_part + at * kDim);
  for (int c = 0; c < chunks; ++c) add(a.e_ws[c * step + at], a.o_ws + (c * step + at) * kDim);
  const float inv = m == -INFINITY ? 0.f : __fdiv_rn(1.f, l);
  const uint2 w = make_uint2(fm::round_pair<T>(o.x * inv, o.y * inv), fm::round_pair<T>(o.z * inv, o.w * inv));
  reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + at * kDim)[lane] = w;
  const float2 x = Elem<T>::to_f2(w.x), y = Elem<T>::to_f2(w.y);
  if (!isfinite(x.x) || !isfinite(x.y) || !isfinite(y.x) || !isfinite(y.y))
    set_status(a.status, NSNKV_ST_OUTPUT_NONFINITE);
  if (a.lse && lane == 0) a.lse[at] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * fm::kLn2;
}

constexpr int kSms = 148;

// Pages per chunk: enough (chunk, head, row tile) CTAs for three per SM.
int chunk_pages_for(int64_t rows, int groups, int G, int h, int32_t max_pages) {
  const int64_t tiles = (rows * G + kRowsCta - 1) / kRowsCta + groups - 1;
  const int64_t units = tiles * h;
  int64_t chunks = (3 * kSms + units - 1) / units;
  if (chunks > max_pages) chunks = max_pages;
  if (chunks < 1) chunks = 1;
  return static_cast<int>((max_pages + chunks - 1) / chunks);
}
int64_t max_chunks(int32_t max_pages, int chunk) { return (max_pages + chunk - 1) / chunk; }

template <int BITS, typename T>
int launch(const PrefixArgs &a, int64_t chunks, cudaStream_t st) {
  if (chunks > 0) {
    auto kern = prefix_rows_kernel<BITS, T>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(PrefixSmem<BITS>)) !=
        cudaSuccess)
      return NSNKV_ERR_CUDA;
    kern<<<dim3(static_cast<unsigned>(chunks), a.h, a.groups * a.row_tiles), 128, sizeof(PrefixSmem<BITS>), st>>>(a);
    if (cudaGetLastError() != cudaSuccess) return NSNKV_ERR_LAUNCH;
  }
  prefix_merge_kernel<T><<<static_cast<unsigned>((a.rows * a.hq + 3) / 4), 128, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

}  // namespace
}  // namespace nsnkv

using namespace nsnkv;

extern "C" {

int64_t nsnkv_prefix_attn_workspace_bytes(int64_t rows, int32_t groups, int hq, int h, int32_t max_pages) {
  if (rows <= 0 || groups <= 0 || hq <= 0 || h <= 0 || hq % h || max_pages < 0) return 0;
  const int64_t chunks = max_pages ? max_chunks(max_pages, chunk_pages_for(rows, groups, hq / h, h, max_pages)) : 0;
  return chunks * rows * hq * (kDim + 1) * 4;
}

int nsnkv_prefix_attn(int64_t rows, int32_t groups, int64_t max_rows, int hq, int h, int bits, int dtype, const void *q,
                      const uint8_t *records, int64_t pages, int64_t rec_stride_head, int64_t rec_stride_page,
                      const int32_t *table, int64_t table_stride, const int32_t *n_pages, int32_t max_pages,
                      const int32_t *row_offsets, const int32_t *row_index, const float *o_part, const float *lse_part,
                      void *out, float *lse, void *workspace, int64_t workspace_bytes, int32_t *status, void *stream) {
  if (rows < 0 || groups <= 0 || max_rows < 0 || hq <= 0 || h <= 0 || hq % h || h > 65535 || max_pages < 0 || pages < 0)
    return NSNKV_ERR_ARG;
  if ((bits != 3 && bits != 5) || (dtype != NSNKV_F16 && dtype != NSNKV_BF16)) return NSNKV_ERR_ARG;
  if (rows == 0) return NSNKV_OK;
  if (groups > 1 && !row_offsets) return NSNKV_ERR_ARG;
  if (!q || !out || !aligned16(q) || !aligned16(out) || (o_part == nullptr) != (lse_part == nullptr) ||
      !aligned16(o_part))
    return NSNKV_ERR_ARG;
  const int64_t rec = 2 * (code_bytes(bits) + 768);
  if (max_pages > 0 && (!records || !table || pages == 0 || !aligned16(records) || rec_stride_head % 16 ||
                        rec_stride_page % 16 || rec_stride_page < rec || table_stride < max_pages))
    return NSNKV_ERR_ARG;
  if (nsnkv_prefix_attn_workspace_bytes(rows, groups, hq, h, max_pages) > workspace_bytes ||
      (max_pages > 0 && (!workspace || !aligned16(workspace))))
    return NSNKV_ERR_ARG;
  if (rows * hq > (int64_t{1} << 32) || groups > 4096) return NSNKV_ERR_TOO_LARGE;
  const int G = hq / h;
  const int chunk = max_pages ? chunk_pages_for(rows, groups, G, h, max_pages) : 1;
  const int64_t chunks = max_pages ? max_chunks(max_pages, chunk) : 0;
  if (max_rows <= 0 || max_rows > rows) max_rows = rows;
  int64_t tiles = (max_rows * G + kRowsCta - 1) / kRowsCta;
  if (tiles * groups > 65535) tiles = 65535 / groups;
  PrefixArgs a{q, records, table, n_pages, row_offsets, row_index, o_part, lse_part, out, lse,
               static_cast<float *>(workspace), static_cast<float *>(workspace) + chunks * rows * hq * kDim,
               rows, pages, table_stride, rec_stride_head, rec_stride_page, groups, hq, h, max_pages, chunk,
               static_cast<int32_t>(tiles), status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bits == 3)
    return dtype == NSNKV_F16 ? launch<3, __half>(a, chunks, st) : launch<3, __nv_bfloat16>(a, chunks, st);
  return dtype == NSNKV_F16 ? launch<5, __half>(a, chunks, st) : launch<5, __nv_bfloat16>(a, chunks, st);
}

}  // extern "C"
