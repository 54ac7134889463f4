// Page operations of a paged cache whose sequences share pages (include/nsnkv.h): fork,
// free, reserve, copy and compact over a block table and per-page reference counts, all on
// the device and in stream order, so a serving loop never reads a table back.
//
// Invariants kept by every operation: refs[p] (p > 0) counts the table entries equal to p;
// page 0 is the unassigned page (a table entry 0 names no page) and refs[0] is left alone.
// Every count is a sum, so the atomics' order does not show in a result.
// The reference has no pages: its caches grow by torch.cat per slot
// (experiments/nb06/source/loop_kv_nb06_packed.py:36-50).
#include "nsnkv_common.cuh"

namespace nsnkv {
namespace {

struct ForkArgs {
  int32_t *table;
  int32_t *n_blocks, *tail_len, *refs;
  uint8_t *k_tail, *v_tail;
  const int32_t *src, *dst;
  int64_t table_stride, tail_seq, tail_head, pages;  // tail strides in bytes
  int32_t batch, h, max_blocks;
  int32_t *status;
};

__device__ __forceinline__ void drop_ref(int32_t *refs, int64_t pages, int32_t page, int32_t *status) {
  if (page == 0) return;
  if (page > 0 && page < pages)
    atomicSub(refs + page, 1);
  else
    set_status(status, NSNKV_ST_PAGE);
}

// Pair i = blockIdx.x.  blockIdx.y == 0: the table row and the counters; otherwise one head of
// the K or V tail, tail_len[src] rows of 256 bytes.  Sources are not targets, so the parts of
// a pair and the pairs are independent.  10 us for 56 targets of eight heads (cold), latency.
__global__ void __launch_bounds__(128) fork_kernel(const ForkArgs a) {
  const int tid = threadIdx.x;
  const int32_t s = a.src[blockIdx.x], d = a.dst[blockIdx.x];
  if (s < 0 || s >= a.batch || d < 0 || d >= a.batch || s == d) {
    if (tid == 0 && blockIdx.y == 0 && s != d) set_status(a.status, NSNKV_ST_PAGE);
    return;
  }
  if (blockIdx.y == 0) {
    const int32_t n = min(max(a.n_blocks[s], 0), a.max_blocks);
    int32_t *from = a.table + s * a.table_stride, *to = a.table + d * a.table_stride;
    for (int i = tid; i < a.max_blocks; i += 128) {
      int32_t next = i < n ? from[i] : 0;
      if (next < 0 || next >= a.pages) {  // names no page of the pool: not handed on
        set_status(a.status, NSNKV_ST_PAGE);
        next = 0;
      }
      drop_ref(a.refs, a.pages, to[i], a.status);
      if (next > 0) atomicAdd(a.refs + next, 1);
      to[i] = next;
    }
    if (tid == 0) {
      a.n_blocks[d] = n;
      a.tail_len[d] = a.tail_len[s];
    }
    return;
  }
  const int part = blockIdx.y - 1, head = part >> 1;
  uint8_t *tail = part & 1 ? a.v_tail : a.k_tail;
  const uint4 *from = reinterpret_cast<const uint4 *>(tail + s * a.tail_seq + head * a.tail_head);
  uint4 *to = reinterpret_cast<uint4 *>(tail + d * a.tail_seq + head * a.tail_head);
  const int n = min(max(a.tail_len[s], 0), kBlock) * (kDim * 2 / 16);
  // at most 8 pieces per thread, all loaded before the first is stored
  uint4 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (tid + 128 * i < n) x[i] = from[tid + 128 * i];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (tid + 128 * i < n) to[tid + 128 * i] = x[i];
}

__global__ void __launch_bounds__(128) free_kernel(const ForkArgs a) {
  const int32_t d = a.dst[blockIdx.x];
  if (d < 0 || d >= a.batch) {
    if (threadIdx.x == 0) set_status(a.status, NSNKV_ST_PAGE);
    return;
  }
  for (int i = threadIdx.x; i < a.max_blocks; i += 128) {
    // the exchange makes a sequence named twice drop its pages once
    drop_ref(a.refs, a.pages, atomicExch(a.table + d * a.table_stride + i, 0), a.status);
  }
  if (threadIdx.x == 0) a.n_blocks[d] = a.tail_len[d] = 0;
}

constexpr int kScan = 1024;

// Exclusive prefix sum of x over the block; total in `sum`.
__device__ __forceinline__ int block_scan(int x, int &sum) {
  __shared__ int part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int y = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) y += up;
  }
  __syncthreads();  // part[] of an earlier scan has been read
  if (lane == 31) part[warp] = y;
  __syncthreads();
  int z = part[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, z, d);
    if (lane >= d) z += up;
  }
  sum = __shfl_sync(0xffffffffu, z, 31);
  const int before = __shfl_sync(0xffffffffu, z, (warp + 31) & 31);
  return y - x + (warp ? before : 0);
}

// Table entries n_blocks[b] .. n_blocks[b] + ahead - 1 that name no page get free pages: the
// entries in (sequence, entry) order take the free pages in ascending order.  One CTA: 12 us a
// call for 64 sequences, most of it the launch and the call.
__global__ void __launch_bounds__(kScan) reserve_kernel(int32_t *table, int64_t table_stride, const int32_t *n_blocks,
                                                        int32_t *refs, int64_t pages, int32_t batch, int32_t max_blocks,
                                                        int32_t ahead, int32_t *status) {
  const int tid = threadIdx.x;
  // each thread owns a run of sequences
  const int per = (batch + kScan - 1) / kScan, b0 = min(tid * per, batch), b1 = min(b0 + per, batch);
  int need = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = min(max(n_blocks[b], 0), max_blocks);
    for (int i = n; i < min(n + ahead, max_blocks); ++i) need += table[b * table_stride + i] <= 0;
  }
  int total;
  const int first = block_scan(need, total);
  if (total == 0) return;
  __shared__ int32_t found[kScan];  // free pages of the current tile, ascending
  int given = 0;                    // free pages handed out by the tiles before
  int taken = 0;                    // of them, to this thread's run (always its first needs)
  for (int64_t base = 1; base < pages && given < total; base += kScan) {
    const int64_t p = base + tid;
    const bool free_page = p < pages && refs[p] <= 0;
    int here;
    const int rank = block_scan(free_page, here);
    if (free_page) {
      found[rank] = static_cast<int32_t>(p);
      if (given + rank < total) refs[p] = 1;
    }
    __syncthreads();
    if (first < given + here && first + need > given) {
      int at = first + taken;
      for (int b = b0; b < b1; ++b) {
        const int n = min(max(n_blocks[b], 0), max_blocks);
        for (int i = n; i < min(n + ahead, max_blocks); ++i) {
          int32_t &e = table[b * table_stride + i];
          if (e > 0) continue;
          if (at >= given + here) break;
          e = found[at - given];
          ++at;
          ++taken;
        }
      }
    }
    __syncthreads();
    given += here;
  }
  if (tid == 0 && given < total) set_status(status, NSNKV_ST_CAPACITY);
}

// Compaction plan.  With L live pages (refs > 0, page 0 counted), the i-th live page at or
// above L moves to the i-th free page below L, both in ascending order: the fewest moves that
// bring the live pages to [0, L), and no destination is a source.  One CTA: the counts are read
// once, coalesced, into a bit per page (bits, before: one word per 32 pages), and ranks come
// from a scan over the words; counting in runs of pages per thread took 26 us for 19201 pages.
__global__ void __launch_bounds__(kScan) compact_plan_kernel(const int32_t *refs, int64_t pages, int32_t *refs_out,
                                                             int32_t *live_out, int32_t *src, int32_t *dst,
                                                             int32_t *map, int32_t *moves, uint32_t *bits,
                                                             int32_t *before) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int words = static_cast<int>((pages + 31) / 32);
#pragma unroll 4
  for (int w = tid >> 5; w < words; w += kScan / 32) {
    const int64_t p = static_cast<int64_t>(w) * 32 + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, p < pages && (p == 0 || refs[p] > 0));
    if (lane == 0) bits[w] = m;
  }
  __syncthreads();
  const int per = (words + kScan - 1) / kScan, w0 = min(tid * per, words), w1 = min(w0 + per, words);
  int n = 0;
  for (int w = w0; w < w1; ++w) n += __popc(bits[w]);
  int live;
  int rank = block_scan(n, live);
  __shared__ int below;  // live pages below L
  if (tid == 0) below = live;
  __syncthreads();
  for (int w = w0; w < w1; ++w) {
    before[w] = rank;
    if (live >> 5 == w) below = rank + __popc(bits[w] & ((1u << (live & 31)) - 1u));
    rank += __popc(bits[w]);
  }
  __syncthreads();
  const int low = below;
  if (tid == 0) {
    *live_out = live;
    *moves = live - low;
  }
#pragma unroll 4
  for (int w = tid >> 5; w < words; w += kScan / 32) {
    const int p = w * 32 + lane;
    const uint32_t m = bits[w];
    const int r = before[w] + __popc(m & ((1u << lane) - 1u));
    const bool used = m >> lane & 1;
    if (p >= pages) continue;
    if (p >= live) {
      if (used)
        src[r - low] = p;
      else
        map[p] = p;
    } else if (!used) {
      dst[p - r] = p;
    }
  }
  __syncthreads();
  // refs_out may be refs: counts move down first, then the pages at or above L are cleared
  for (int i = tid; i < live - low; i += kScan) {
    const int s = src[i], d = dst[i];
    map[s] = d;
    refs_out[d] = refs[s];
  }
  __syncthreads();
#pragma unroll 4
  for (int64_t p = tid; p < pages; p += kScan) {
    if (p >= live)
      refs_out[p] = 0;
    else if (bits[p >> 5] >> (p & 31) & 1)
      refs_out[p] = refs[p];
  }
}

struct MoveArgs {
  nsnkv_page_array arr[NSNKV_MAX_PAGE_ARRAYS];
  int32_t arrays, h;
  int64_t pages;
  const int32_t *src, *dst, *count;  // count: device (null: max_count)
  int32_t max_count;
  // table remap (null: none): entries >= *live take map[entry]
  const int32_t *table, *map, *live;
  int32_t *table_out;
  int64_t table_rows, table_cols, table_stride, out_stride;
  int32_t *status;
};

// Work item (move i, head j): the page's bytes of every array in 16-byte pieces, kPieces per
// thread and round, all loaded before the first is stored (a page is at most a few KB: one or
// two rounds).  The next item's page numbers are read while an item is copied.  4800 pages of
// eight heads, INT3 (610 MB read and written): 138 us with the plan, 4.4 TB/s (timed apart: move
// 109 us, plan 20 us); with the loads and stores of a piece in turn it was 192 us.
constexpr int kMoveThreads = 128, kPieces = 4;
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MoveArgs a) {
  const int tid = threadIdx.x;
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * kMoveThreads + tid;
  if (a.table) {
    const int32_t live = *a.live;
    for (int64_t e = gid; e < a.table_rows * a.table_cols; e += static_cast<int64_t>(gridDim.x) * kMoveThreads) {
      const int64_t r = e / a.table_cols, c = e % a.table_cols;
      int32_t t = a.table[r * a.table_stride + c];
      if (t >= a.pages || t < 0)
        set_status(a.status, NSNKV_ST_PAGE);
      else if (t >= live)
        t = a.map[t];
      a.table_out[r * a.out_stride + c] = t;
    }
  }
  const int64_t items = static_cast<int64_t>(a.count ? *a.count : a.max_count) * a.h;
  int total = 0;
  for (int x = 0; x < a.arrays; ++x) total += static_cast<int>(a.arr[x].bytes / 16);
  int64_t item = blockIdx.x;
  int32_t s = 0, d = 0;
  if (item < items) s = a.src[item / a.h], d = a.dst[item / a.h];
  while (item < items) {
    const int64_t j = item % a.h, next = item + gridDim.x;
    int32_t s_next = 0, d_next = 0;
    if (next < items) s_next = a.src[next / a.h], d_next = a.dst[next / a.h];
    if (s < 0 || s >= a.pages || d < 0 || d >= a.pages) {
      if (tid == 0) set_status(a.status, NSNKV_ST_PAGE);
    } else {
      for (int u0 = 0; u0 < total; u0 += kMoveThreads * kPieces) {
        uint4 v[kPieces], *to[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          int u = u0 + i * kMoveThreads + tid, x = 0;
          to[i] = nullptr;
          if (u >= total) continue;
          while (u >= a.arr[x].bytes / 16) u -= static_cast<int>(a.arr[x++].bytes / 16);
          uint8_t *head = static_cast<uint8_t *>(a.arr[x].base) + j * a.arr[x].stride_head;
          to[i] = reinterpret_cast<uint4 *>(head + d * a.arr[x].stride_page) + u;
          v[i] = __ldcs(reinterpret_cast<const uint4 *>(head + s * a.arr[x].stride_page) + u);
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          if (to[i]) __stcs(to[i], v[i]);
      }
    }
    item = next, s = s_next, d = d_next;
  }
}

int check_arrays(int h, int64_t pages, int arrays, const nsnkv_page_array *arr) {
  if (h <= 0 || pages <= 0 || arrays < 0 || arrays > NSNKV_MAX_PAGE_ARRAYS || (arrays > 0 && !arr)) return NSNKV_ERR_ARG;
  for (int x = 0; x < arrays; ++x)
    if (!arr[x].base || !aligned16(arr[x].base) || arr[x].bytes <= 0 || arr[x].bytes % 16 || arr[x].stride_page % 16 ||
        arr[x].stride_head % 16 || arr[x].bytes > (int64_t{1} << 30))
      return NSNKV_ERR_ARG;
  return NSNKV_OK;
}

// CTAs of the move kernel: twelve per SM, each with a page's loads in flight.
constexpr int kMoveCtas = 148 * 12;

}  // namespace
}  // namespace nsnkv

using namespace nsnkv;

extern "C" {

int nsnkv_fork_sequences(int64_t batch, int h, int64_t pages, int32_t *block_table, int64_t table_stride,
                         int32_t max_blocks, int32_t *n_blocks, int32_t *tail_len, int32_t *page_refs, void *k_tail,
                         void *v_tail, int64_t tail_stride_seq, int64_t tail_stride_head, int64_t count,
                         const int32_t *src, const int32_t *dst, int32_t *status, void *stream) {
  if (batch <= 0 || batch > INT32_MAX || h <= 0 || h > 32767 || pages <= 0 || max_blocks <= 0 ||
      table_stride < max_blocks || count < 0 || count > INT32_MAX)
    return NSNKV_ERR_ARG;
  if (count == 0) return NSNKV_OK;
  if (!block_table || !n_blocks || !tail_len || !page_refs || !k_tail || !v_tail || !src || !dst) return NSNKV_ERR_ARG;
  if (!aligned16(k_tail) || !aligned16(v_tail) || tail_stride_head < kBlock || tail_stride_seq < kBlock)
    return NSNKV_ERR_ARG;
  const ForkArgs a{block_table, n_blocks, tail_len, page_refs, static_cast<uint8_t *>(k_tail),
                   static_cast<uint8_t *>(v_tail), src, dst, table_stride, tail_stride_seq * kDim * 2,
                   tail_stride_head * kDim * 2, pages, static_cast<int32_t>(batch), h, max_blocks, status};
  fork_kernel<<<dim3(static_cast<unsigned>(count), 1 + 2 * h), 128, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

int nsnkv_free_sequences(int64_t batch, int64_t pages, int32_t *block_table, int64_t table_stride, int32_t max_blocks,
                         int32_t *n_blocks, int32_t *tail_len, int32_t *page_refs, int64_t count, const int32_t *seqs,
                         int32_t *status, void *stream) {
  if (batch <= 0 || batch > INT32_MAX || pages <= 0 || max_blocks <= 0 || table_stride < max_blocks || count < 0 ||
      count > INT32_MAX)
    return NSNKV_ERR_ARG;
  if (count == 0) return NSNKV_OK;
  if (!block_table || !n_blocks || !tail_len || !page_refs || !seqs) return NSNKV_ERR_ARG;
  ForkArgs a{};
  a.table = block_table;
  a.n_blocks = n_blocks;
  a.tail_len = tail_len;
  a.refs = page_refs;
  a.dst = seqs;
  a.table_stride = table_stride;
  a.pages = pages;
  a.batch = static_cast<int32_t>(batch);
  a.max_blocks = max_blocks;
  a.status = status;
  free_kernel<<<static_cast<unsigned>(count), 128, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

int nsnkv_reserve_pages(int64_t batch, int64_t pages, int32_t *block_table, int64_t table_stride, int32_t max_blocks,
                        const int32_t *n_blocks, int32_t *page_refs, int32_t ahead, int32_t *status, void *stream) {
  if (batch <= 0 || batch > (1 << 20) || pages <= 0 || pages > INT32_MAX || max_blocks <= 0 ||
      table_stride < max_blocks || ahead < 0 || ahead > max_blocks)
    return NSNKV_ERR_ARG;
  if (!block_table || !n_blocks || !page_refs) return NSNKV_ERR_ARG;
  if (batch * ahead > INT32_MAX) return NSNKV_ERR_TOO_LARGE;  // the kernel counts entries in 32 bits
  reserve_kernel<<<1, kScan, 0, static_cast<cudaStream_t>(stream)>>>(block_table, table_stride, n_blocks, page_refs,
                                                                     pages, static_cast<int32_t>(batch), max_blocks,
                                                                     ahead, status);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

int nsnkv_copy_pages(int h, int64_t pages, int arrays, const nsnkv_page_array *arr, int64_t count, const int32_t *src,
                     const int32_t *dst, int32_t *status, void *stream) {
  if (count < 0 || count > INT32_MAX || pages > INT32_MAX) return NSNKV_ERR_ARG;
  if (const int rc = check_arrays(h, pages, arrays, arr)) return rc;
  if (count == 0 || arrays == 0) return NSNKV_OK;
  if (!src || !dst) return NSNKV_ERR_ARG;
  MoveArgs a{};
  for (int x = 0; x < arrays; ++x) a.arr[x] = arr[x];
  a.arrays = arrays;
  a.h = h;
  a.pages = pages;
  a.src = src;
  a.dst = dst;
  a.max_count = static_cast<int32_t>(count);
  a.status = status;
  const int64_t items = count * h;
  move_kernel<<<static_cast<unsigned>(items < kMoveCtas ? items : kMoveCtas), kMoveThreads, 0,
                static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

int64_t nsnkv_compact_pages_workspace_bytes(int64_t pages) { return pages > 0 ? (3 * pages + 2 + 2 * ((pages + 31) / 32)) * 4 : 0; }

int nsnkv_compact_pages(int h, int64_t pages, int arrays, const nsnkv_page_array *arr, int64_t batch,
                        int32_t max_blocks, const int32_t *block_table, int64_t table_stride, int32_t *table_out,
                        int64_t table_out_stride, const int32_t *page_refs, int32_t *refs_out, int32_t *live,
                        void *workspace, int64_t workspace_bytes, int32_t *status, void *stream) {
  if (pages > INT32_MAX || batch < 0 || max_blocks < 0 || table_stride < max_blocks || table_out_stride < max_blocks)
    return NSNKV_ERR_ARG;
  if (const int rc = check_arrays(h, pages, arrays, arr)) return rc;
  if (!page_refs || !refs_out || !live || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
      workspace_bytes < nsnkv_compact_pages_workspace_bytes(pages) ||
      (batch > 0 && max_blocks > 0 && (!block_table || !table_out)))
    return NSNKV_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t *src = static_cast<int32_t *>(workspace), *dst = src + pages, *map = dst + pages, *moves = map + pages;
  int32_t *bits = moves + 1, *before = bits + (pages + 31) / 32;
  compact_plan_kernel<<<1, kScan, 0, st>>>(page_refs, pages, refs_out, live, src, dst, map, moves,
                                           reinterpret_cast<uint32_t *>(bits), before);
  if (cudaGetLastError() != cudaSuccess) return NSNKV_ERR_LAUNCH;
  MoveArgs a{};
  for (int x = 0; x < arrays; ++x) a.arr[x] = arr[x];
  a.arrays = arrays;
  a.h = h;
  a.pages = pages;
  a.src = src;
  a.dst = dst;
  a.count = moves;
  if (batch > 0 && max_blocks > 0) {
    a.table = block_table;
    a.table_out = table_out;
    a.map = map;
    a.live = live;
    a.table_rows = batch;
    a.table_cols = max_blocks;
    a.table_stride = table_stride;
    a.out_stride = table_out_stride;
  }
  a.status = status;
  const int64_t most = (pages / 2 + 1) * h;
  move_kernel<<<static_cast<unsigned>(most < kMoveCtas ? most : kMoveCtas), kMoveThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

}  // extern "C"
