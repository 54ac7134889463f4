// Causal attention over whole prompts packed one after another (include/nsnkv.h,
// nsnkv_prompt_attn): grouped heads, sequences of different lengths.
//
// The reference runs a prompt through the model's own attention (the OFFICIAL arm of
// experiments/nb06/source/loop_kv_nb06_attention.py:33-88) before its cache compresses the
// keys and values; this is that attention for a packed batch, without repeated K / V heads
// and without padding.
#include "flash_mma.cuh"
#include "prompt_tc.cuh"

namespace nsnkv {
namespace {

struct PromptArgs {
  const void *q, *k, *v;
  void *out;
  float *lse;
  const int32_t *cu;
  int64_t tokens;
  int64_t q_tok, q_head, kv_tok, kv_head, v_tok, v_head;  // strides in elements
  int32_t seqs, hq, h, causal;
  int32_t *status;
};

// Sequence s of the packed batch as token indices inside [0, tokens).
__device__ __forceinline__ void seq_range(const PromptArgs &a, int s, int64_t &begin, int64_t &end) {
  begin = min(max(static_cast<int64_t>(a.cu[s]), int64_t{0}), a.tokens);
  end = min(max(static_cast<int64_t>(a.cu[s + 1]), begin), a.tokens);
}

constexpr int kSms = 148;
constexpr int kRowsCta = 64;
struct RowsSmem {
  uint16_t k[2][fm::kTile][fm::kRow];
  uint16_t v[2][fm::kTile][fm::kRow];
};

__device__ __forceinline__ void cp16(void *dst, const void *src, bool in) {
  const int n = in ? 16 : 0;  // 0: the 16 bytes are zero-filled and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(n)
               : "memory");
}

// Short prompts (mma.sync): latency bound, 7 us on the device for 3 prompts of 59 tokens in all;
// 325 us for 4 x 2048 tokens of 16 heads, where the tensor-core kernel takes 98 us.
// 64 query rows of one head per CTA, 16 per warp; K / V tiles of 64 tokens double-buffered
// with cp.async.  Tokens past the sequence are zero-filled, so another sequence's values
// never enter a product.
template <typename T>
__global__ void __launch_bounds__(128, 3) prompt_rows_kernel(const PromptArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  RowsSmem &S = *reinterpret_cast<RowsSmem *>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y, kvh = head / (a.hq / a.h);
  int64_t begin, end;
  seq_range(a, blockIdx.z, begin, end);
  const int64_t len = end - begin;
  const T *kb = static_cast<const T *>(a.k) + begin * a.kv_tok + kvh * a.kv_head;
  const T *vb = static_cast<const T *>(a.v) + begin * a.v_tok + kvh * a.v_head;

  for (int64_t qt = blockIdx.x; qt * kRowsCta < len; qt += gridDim.x) {
    const int64_t row0 = qt * kRowsCta;
    const int64_t r0 = row0 + 16 * warp + (lane >> 2), r1 = r0 + 8;  // this lane's rows
    const T *qb = static_cast<const T *>(a.q) + begin * a.q_tok + head * a.q_head;
    fm::Rows st;
    st.init();
    st.load_q<T>(r0 < len ? qb + r0 * a.q_tok : nullptr, r1 < len ? qb + r1 * a.q_tok : nullptr, lane);
    const int64_t keys = a.causal ? min(len, row0 + kRowsCta) : len;
    const int tiles = static_cast<int>((keys + fm::kTile - 1) / fm::kTile);
    auto load = [&](int tile) {
      const int buf = tile & 1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = tid + 128 * i, r = e >> 4, c = (e & 15) * 8;
        const int64_t tok = static_cast<int64_t>(tile) * fm::kTile + r;
        const bool in = tok < len;
        const int64_t at = in ? tok : 0;
        cp16(&S.k[buf][r][c], kb + at * a.kv_tok + c, in);
        cp16(&S.v[buf][r][c], vb + at * a.v_tok + c, in);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();  // the previous row tile is done with the buffers
    load(0);
    for (int tile = 0; tile < tiles; ++tile) {
      if (tile + 1 < tiles) load(tile + 1);
      if (tile + 1 < tiles)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
      const int64_t t0 = static_cast<int64_t>(tile) * fm::kTile;
      // row r sees the tokens up to r (causal), up to the end otherwise
      const int64_t lim0 = (a.causal ? min(len, r0 + 1) : len) - t0, lim1 = (a.causal ? min(len, r1 + 1) : len) - t0;
      const int n0 = static_cast<int>(max(min(lim0, int64_t{fm::kTile}), int64_t{0}));
      const int n1 = static_cast<int>(max(min(lim1, int64_t{fm::kTile}), int64_t{0}));
      const int buf = tile & 1;
      // A non-finite value of a token that some rows do not see must not reach them through
      // a product with p = 0: in the tiles on the diagonal such tokens' V rows are taken out
      // of the product and added by the rows that do see them.
      int bad = 0;
      if (a.causal && t0 + fm::kTile > row0 + 1) {
        const uint32_t *vr = reinterpret_cast<const uint32_t *>(&S.v[buf][tid >> 1][(tid & 1) * 64]);
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
          const float2 x = Elem<T>::to_f2(vr[i]);
          bad |= !isfinite(x.x) || !isfinite(x.y);
        }
        bad = __syncthreads_or(bad);
      }
      if (bad)
        st.tile_guarded<T>(S.k[buf], S.v[buf], n0, n1, lane);
      else
        st.tile<T>(S.k[buf], S.v[buf], n0, n1, lane);
      __syncthreads();  // every warp is done with this buffer before it is loaded again
    }
    float inv[2];
    st.finish(inv);
    int nonfinite = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = i ? r1 : r0;
      if (r >= len) continue;
      T *orow = static_cast<T *>(a.out) + ((begin + r) * a.hq + head) * kDim;
#pragma unroll
      for (int nt = 0; nt < 16; ++nt) {
        const uint32_t w = fm::round_pair<T>(st.o[nt][2 * i] * inv[i], st.o[nt][2 * i + 1] * inv[i]);
        reinterpret_cast<uint32_t *>(orow)[4 * nt + (lane & 3)] = w;
        const float2 x = Elem<T>::to_f2(w);
        nonfinite |= !isfinite(x.x) || !isfinite(x.y);
      }
      if (a.lse && (lane & 3) == 0) a.lse[(begin + r) * a.hq + head] = st.lse2(i) * fm::kLn2;
    }
    if (nonfinite) set_status(a.status, NSNKV_ST_OUTPUT_NONFINITE);
  }
}

template <typename T>
int launch_rows(const PromptArgs &a, int64_t longest, cudaStream_t st) {
  auto kern = prompt_rows_kernel<T>;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kern, sizeof(RowsSmem), done)) return NSNKV_ERR_CUDA;
  const int64_t tiles = (longest + kRowsCta - 1) / kRowsCta;
  const dim3 grid(static_cast<unsigned>(tiles < 65535 ? tiles : 65535), a.hq, a.seqs);
  kern<<<grid, 128, sizeof(RowsSmem), st>>>(a);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

// Tensor map of x [tokens][heads][128] with element strides: boxes of 64 channels of one
// head and 128 tokens, 128-byte swizzle.
bool make_map(CUtensorMap *map, const void *base, int dtype, int64_t tokens, int heads, int64_t tok, int64_t head) {
  static const auto encode = [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult got;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &got) != cudaSuccess ||
        got != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn);
  }();
  if (!encode) return false;
  const cuuint64_t dims[3] = {kDim, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  // the stride of a dimension of one element is never used
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? head : kDim) * 2,
                                 static_cast<cuuint64_t>(tokens > 1 ? tok : kDim) * 2};
  const cuuint32_t box[3] = {64, 1, ptc::kN}, step[3] = {1, 1, 1};
  return encode(map, dtype == NSNKV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
int launch_tc(const PromptArgs &p, int dtype, cudaStream_t st) {
  ptc::Maps maps;
  if (!make_map(&maps.q, p.q, dtype, p.tokens, p.hq, p.q_tok, p.q_head) ||
      !make_map(&maps.k, p.k, dtype, p.tokens, p.h, p.kv_tok, p.kv_head) ||
      !make_map(&maps.v, p.v, dtype, p.tokens, p.h, p.v_tok, p.v_head))
    return NSNKV_ERR_CUDA;
  const ptc::Args a{p.cu, p.out, p.lse, p.q, p.k, p.v, p.tokens, p.q_tok, p.q_head, p.kv_tok, p.kv_head, p.v_tok,
                    p.v_head, p.seqs, p.hq, p.h, p.causal, p.status};
  auto kern = ptc::prompt_tc_kernel<T>;
  const int smem = static_cast<int>(sizeof(ptc::Smem)) + 1024;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kern, smem, done)) return NSNKV_ERR_CUDA;
  // at most one pair of row tiles per 256 tokens and one more per sequence
  const int64_t items = (p.tokens / (2 * ptc::kM) + p.seqs) * p.hq;
  kern<<<static_cast<unsigned>(items < kSms ? items : kSms), ptc::kThreads, smem, st>>>(a, maps);
  return cudaGetLastError() == cudaSuccess ? NSNKV_OK : NSNKV_ERR_LAUNCH;
}

}  // namespace
}  // namespace nsnkv

using namespace nsnkv;

extern "C" int nsnkv_prompt_attn(int64_t tokens, int32_t seqs, int64_t longest, int hq, int h, int dtype, int causal,
                                 const void *q, int64_t q_tok, int64_t q_head, const void *k, int64_t k_tok,
                                 int64_t k_head, const void *v, int64_t v_tok, int64_t v_head, const int32_t *cu_seqlens,
                                 void *out, float *lse, int32_t *status, void *stream) {
  if (tokens < 0 || seqs < 0 || seqs > 65535 || longest < 0 || hq <= 0 || h <= 0 || hq % h || hq > 65535)
    return NSNKV_ERR_ARG;
  if (dtype != NSNKV_F16 && dtype != NSNKV_BF16) return NSNKV_ERR_ARG;
  if (tokens == 0 || seqs == 0) return NSNKV_OK;
  if (!q || !k || !v || !cu_seqlens || !out || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return NSNKV_ERR_ARG;
  for (int64_t s : {q_tok, q_head, k_tok, k_head, v_tok, v_head})
    if (s < 0 || s % 8) return NSNKV_ERR_ARG;
  PromptArgs a{q, k, v, out, lse, cu_seqlens, tokens, q_tok, q_head, k_tok, k_head, v_tok, v_head, seqs, hq, h,
               causal != 0, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (longest == 0 || longest > tokens) longest = tokens;  // 0: not known
  if (tokens > INT32_MAX || (tokens / 256 + seqs) * hq > INT32_MAX) return NSNKV_ERR_TOO_LARGE;
  // The tensor-core kernel from 65 rows on: 16 sequences of 64 tokens, GQA 32:8, take 18.3 us here and
  // 19.9 us there, of 128 tokens 33.0 and 21.8 us, of 256 tokens 72.6 and 36.2 us.  Its stores are
  // 32 bytes wide, and its tensor maps take no broadcast dimension (a stride of 0).
  const bool broadcast = (hq > 1 && !q_head) || (h > 1 && (!k_head || !v_head)) || (tokens > 1 && (!q_tok || !k_tok || !v_tok));
  if (longest > 64 && !broadcast && (reinterpret_cast<uintptr_t>(out) & 31) == 0)
    return dtype == NSNKV_F16 ? launch_tc<__half>(a, dtype, st) : launch_tc<__nv_bfloat16>(a, dtype, st);
  return dtype == NSNKV_F16 ? launch_rows<__half>(a, longest, st) : launch_rows<__nv_bfloat16>(a, longest, st);
}
