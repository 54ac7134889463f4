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
#include "prefix_tc.cuh"
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

// One warp per (query row, head): the chunks of its group and its own partial.  Lane c holds
// chunk c's log-sum-exp; the chunks' rows are read four at a time.  A part with log-sum-exp -inf
// holds nothing and is left out; one with NaN makes the row NaN (the sum of weights l becomes NaN,
// while the maximum passes NaN over).
template <typename T>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the chunk kernel runs
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (item >= a.rows * a.hq) return;
  const uint32_t hq = a.hq, p = static_cast<uint32_t>(item) / hq, head = static_cast<uint32_t>(item) - p * hq;
  const int64_t r = row_at(a, p);
  if (r < 0) return;
  int chunks = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    int64_t begin = 0, end = 0;
    if (g0 + lane < a.groups) group_rows(a, g0 + lane, begin, end);
    const bool in = p >= begin && p < end;
    const int n = in ? (group_pages(a, g0 + lane) + a.chunk_pages - 1) / a.chunk_pages : 0;
    chunks = max(chunks, __reduce_max_sync(0xffffffffu, n));
  }
  const int64_t at = r * a.hq + head, step = a.rows * a.hq;
  const float own = a.lse_part ? a.lse_part[at] * fm::kLog2e : -INFINITY;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (own != -INFINITY) o = reinterpret_cast<const float4 *>(a.o_part + at * kDim)[lane];  // else it is not read
  float m = own, l = own == -INFINITY ? 0.f : isnan(own) ? own : 1.f;
  for (int c0 = 0; c0 < chunks; c0 += 32) {
    const float e = c0 + lane < chunks ? a.e_ws[(c0 + lane) * step + at] : -INFINITY;
    float top = e;
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new;
    const float w = e == -INFINITY ? 0.f : fm::ex2(e - base), c = m == -INFINITY ? 0.f : fm::ex2(m - base);
    float sum = w;
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * c + sum;
    o.x *= c, o.y *= c, o.z *= c, o.w *= c;
    m = m_new;
    const int n = min(32, chunks - c0);
    for (int i = 0; i < n; i += 4) {
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) x[k] = reinterpret_cast<const float4 *>(a.o_ws + ((c0 + i + k) * step + at) * kDim)[lane];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float wk = __shfl_sync(0xffffffffu, w, (i + k) & 31);
        if (i + k < n && wk != 0.f) {  // 0: the chunk holds nothing for the row (NaN passes)
          o.x += wk * x[k].x;
          o.y += wk * x[k].y;
          o.z += wk * x[k].z;
          o.w += wk * x[k].w;
        }
      }
    }
  }
  const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
  const uint2 w = make_uint2(fm::round_pair<T>(o.x * inv, o.y * inv), fm::round_pair<T>(o.z * inv, o.w * inv));
  reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + at * kDim)[lane] = w;
  const float2 x = Elem<T>::to_f2(w.x), y = Elem<T>::to_f2(w.y);
  if (!isfinite(x.x) || !isfinite(x.y) || !isfinite(y.x) || !isfinite(y.y))
    set_status(a.status, NSNKV_ST_OUTPUT_NONFINITE);
  if (a.lse && lane == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * fm::kLn2;
}

constexpr int kSms = 148;
constexpr int kPairRows = 2 * xtc::kM;

// Pages per chunk.  The kernel runs one CTA per SM and (chunk, head, pair of row tiles); a CTA
// costs about its pages plus five for its start, its partial rows and their merge.
int chunk_pages_for(int64_t rows, int groups, int G, int h, int32_t max_pages) {
  const int64_t units = ((rows * G + kPairRows - 1) / kPairRows + groups - 1) * h;
  int64_t best = max_pages, best_cost = INT64_MAX;
  for (int64_t chunks = 1; chunks <= kSms && chunks <= max_pages; ++chunks) {
    const int64_t per = (max_pages + chunks - 1) / chunks, waves = (units * ((max_pages + per - 1) / per) + kSms - 1) / kSms;
    const int64_t cost = waves * (per + 5);
    if (cost < best_cost) best = per, best_cost = cost;
  }
  return static_cast<int>(best < 1 ? 1 : best);
}
int64_t max_chunks(int32_t max_pages, int chunk) { return (max_pages + chunk - 1) / chunk; }

template <int BITS, typename T>
int launch(const PrefixArgs &a, int64_t chunks, cudaStream_t st) {
  if (chunks > 0) {
    auto kern = xtc::prefix_tc_kernel<BITS, T>;
    const int smem = static_cast<int>(sizeof(xtc::Smem<BITS>)) + 1024;
    static std::atomic<uint64_t> done{0};
    if (!allow_smem(kern, smem, done)) return NSNKV_ERR_CUDA;
    const xtc::Args x{a.q, a.records, a.table, a.n_pages, a.row_offsets, a.row_index, a.o_ws, a.e_ws, a.rows, a.pages,
                      a.table_stride, a.rec_head, a.rec_page, a.hq, a.h, a.max_pages, a.chunk_pages, a.row_tiles,
                      a.status};
    kern<<<dim3(static_cast<unsigned>(chunks), a.h, a.groups * a.row_tiles), xtc::kThreads, smem, st>>>(x);
    if (cudaGetLastError() != cudaSuccess) return NSNKV_ERR_LAUNCH;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((a.rows * a.hq + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = chunks > 0 ? 1 : 0;  // only behind the chunk kernel, which announces it
  return cudaLaunchKernelEx(&cfg, prefix_merge_kernel<T>, a) == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
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
  if (rows * hq > INT32_MAX || groups > 4096) return NSNKV_ERR_TOO_LARGE;
  const int G = hq / h;
  const int chunk = max_pages ? chunk_pages_for(rows, groups, G, h, max_pages) : 1;
  const int64_t chunks = max_pages ? max_chunks(max_pages, chunk) : 0;
  if (max_rows <= 0 || max_rows > rows) max_rows = rows;
  int64_t tiles = (max_rows * G + kPairRows - 1) / kPairRows;
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
