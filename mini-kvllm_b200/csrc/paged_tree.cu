// Attention of trees of drafted tokens over the paged KV cache (speculative decoding).
//
// Sequence b holds len_b cached tokens, the last n_b of them the nodes of its tree; query
// row i of the sequence (node i) attends to the whole prefix t < len_b - n_b and to the
// nodes whose bit its mask row sets:
//   out[i, h] = sum_t p_t V[t] / sum_t p_t,  p_t = exp(scale q[i, h].K[t] - max)
// in fp32, K/V gathered through the block table and dequantised on load, kv head
// h / (H / KVH). A row that sees nothing gives zeros. Tokens on missing pages are skipped.
// What a row does not see never reaches it, be it infinite or NaN.
//
// All query rows of a kv head (nodes x GQA group) share each K/V tile, and the token axis
// is split evenly over the CTAs (paged_tree.cuh), so K and V are read about once.
#include <atomic>

#include "paged_tree.cuh"
#include "sm100.cuh"

namespace mkv {
namespace tree {
namespace {

// ============================================================ CUDA-core kernel
// Every type and head_dim (a multiple of 16, at most 256): 16 rows x 32 tokens per step in
// fp32. A warp owns 4 rows; lane = token for the scores, lane = column for the products. Bound by
// shared memory (5 16-byte loads to 16 products a lane) and, with few rows, by the latency of a
// tile, which four CTAs an SM cover: fp32, 8 sequences of 3-4k tokens, 16 to 32 rows on each of 8 kv
// heads 418 us (2 CTAs: 725); 8 x 4k tokens, 32 rows on each 509 us, 13 times what its bytes take.
// 8 rows a warp have fewer loads per product, but their registers halve the CTAs (479 for 418).
constexpr int kGRows = 16, kGKT = 32, kGThreads = 128;
constexpr int kGCtas = 4 * kNumSMs;  // resident with head_dim up to 128

template <typename CT> __device__ __forceinline__ float elem_f32(const uint8_t* p, int i) {
  return to_f32(reinterpret_cast<const CT*>(p)[i]);
}

template <typename QT, typename CT>
__global__ void __launch_bounds__(kGThreads) paged_tree_generic_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float sm[];
  const int D = p.head_dim, DK = D + 4;
  float* q_sm = sm;                    // [16][D]
  float* k_sm = q_sm + kGRows * D;     // [32][D + 4]
  float* v_sm = k_sm + kGKT * DK;      // [32][D]
  float* p_sm = v_sm + kGKT * D;       // [warp][32 tokens][4 rows]
  float* ks_sm = p_sm + kGRows * kGKT; // [32]
  __shared__ uint32_t page_ok;
  __shared__ long long scratch[kBeginWords(kGThreads)];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kVec = 16 / (int)sizeof(CT);
  const bool per_token = p.k_scales != nullptr;
  const float kst = p.k_scale ? __ldg(p.k_scale) : 1.0f, vst = p.v_scale ? __ldg(p.v_scale) : 1.0f;
  Walk w;
  if (!begin<kGRows, kGKT, kGThreads>(p, blockIdx.x, gridDim.x, scratch, w)) return;
  Unit u;
  while (next<kGRows, kGKT>(p, w, u)) {
    const int rows = min(kGRows, u.s.nodes * p.group - u.mt * kGRows);
    __syncthreads();
    for (int i = tid; i < kGRows * D; i += kGThreads) {
      const int r = i / D, d = i - r * D, R = u.mt * kGRows + r, node = R / p.group;
      q_sm[i] = r < rows ? to_f32(reinterpret_cast<const QT*>(p.q)[(u.s.q0 + node) * p.q_st +
                                 (int64_t)(u.kvh * p.group + R - node * p.group) * p.q_sh + d]) : 0.0f;
    }
    float m[4], l[4], acc[4][8];
    const uint64_t* mrow[4];
    uint64_t m0[4];
    bool any[4];  // whether the row has seen a token
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
      any[r] = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[r][i] = 0.0f;
      const int R = u.mt * kGRows + min(4 * warp + r, rows - 1);
      mrow[r] = p.mask + (u.s.q0 + R / p.group) * p.mask_st;
      m0[r] = __ldg(mrow[r]);
    }
    for (int it = u.k0; it < u.k1; ++it) {
      const int t0 = it * kGKT;
      __syncthreads();  // the previous tile is read
      if (tid < 32) {
        bool ok = false;
        if (t0 + tid < u.s.len) ok = load_page(p, u.b, (t0 + tid) / p.block_size) >= 0;
        const uint32_t v = __ballot_sync(0xffffffffu, ok);
        if (tid == 0) page_ok = v;
      }
      for (int i = tid; i < kGKT * (D / kVec); i += kGThreads) {
        const int t = i / (D / kVec), c = i - t * (D / kVec);
        float* kd = k_sm + t * DK + c * kVec;
        float* vd = v_sm + t * D + c * kVec;
        int64_t page = -1;
        int blk = 0;
        if (t0 + t < u.s.len) {
          blk = (t0 + t) / p.block_size;
          page = load_page(p, u.b, blk);
        }
        if (page >= 0) {
          const int64_t row = (page * p.block_size + (t0 + t - blk * p.block_size)) * p.num_kv_heads + u.kvh;
          const uint4 kr = ld_stream_v4(p.k_cache + (row * D + c * kVec) * (int64_t)sizeof(CT));
          const uint4 vr = ld_stream_v4(p.v_cache + (row * D + c * kVec) * (int64_t)sizeof(CT));
          const float vs = per_token ? __ldg(p.v_scales + row) : vst;
          if (c == 0) ks_sm[t] = per_token ? __ldg(p.k_scales + row) : kst;
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            kd[e] = elem_f32<CT>(reinterpret_cast<const uint8_t*>(&kr), e);
            vd[e] = elem_f32<CT>(reinterpret_cast<const uint8_t*>(&vr), e) * vs;
          }
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e) kd[e] = vd[e] = 0.0f;
          if (c == 0) ks_sm[t] = 0.0f;
        }
      }
      __syncthreads();
      // scores of 4 rows, one token a lane
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const float* kr = k_sm + lane * DK;
      const float* qr = q_sm + 4 * warp * D;
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 qv = *reinterpret_cast<const float4*>(qr + r * D + d);
          s[r] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[r]))));
        }
      }
      const float sc = p.qk_scale_log2 * ks_sm[lane];
      float pr[4], alpha[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t vis = visible32(u.s, mrow[r], m0[r], p.mask_words, t0) & page_ok;
        any[r] |= vis != 0;
        const bool on = (vis >> lane) & 1;
        const float x = on ? s[r] * sc : -INFINITY;
        const float mn = fmaxf(m[r], warp_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn;
        alpha[r] = exp2f(m[r] - base);
        pr[r] = on ? exp2f(x - base) : 0.0f;
        l[r] = fmaf(l[r], alpha[r], warp_sum(pr[r]));
        m[r] = mn;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r][i] *= alpha[r];
      }
      float4* pw = reinterpret_cast<float4*>(p_sm + warp * 4 * kGKT);
      pw[lane] = make_float4(pr[0], pr[1], pr[2], pr[3]);
      __syncwarp();
      // a hidden node's values may be infinite or NaN: they are left out, not multiplied by 0
      const bool hidden = t0 + kGKT > u.s.prefix;
#pragma unroll 4
      for (int t = 0; t < kGKT; ++t) {
        const float4 pv = pw[t];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = lane + 32 * i;
          if (d >= D) break;
          const float v = v_sm[t * D + d];
          if (hidden) {
            acc[0][i] = pv.x == 0.0f ? acc[0][i] : fmaf(pv.x, v, acc[0][i]);
            acc[1][i] = pv.y == 0.0f ? acc[1][i] : fmaf(pv.y, v, acc[1][i]);
            acc[2][i] = pv.z == 0.0f ? acc[2][i] : fmaf(pv.z, v, acc[2][i]);
            acc[3][i] = pv.w == 0.0f ? acc[3][i] : fmaf(pv.w, v, acc[3][i]);
          } else {
            acc[0][i] = fmaf(pv.x, v, acc[0][i]);
            acc[1][i] = fmaf(pv.y, v, acc[1][i]);
            acc[2][i] = fmaf(pv.z, v, acc[2][i]);
            acc[3][i] = fmaf(pv.w, v, acc[3][i]);
          }
        }
      }
      __syncwarp();
    }
    const int slot = slot_of(u, blockIdx.x);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * warp + r;
      if (row >= rows) continue;
      // scores that are all -inf have no softmax (0 / 0); a row that sees nothing is 0
      if (slot < 0) {
        if (l[r] == 0.0f && any[r]) l[r] = NAN;
        const int R = u.mt * kGRows + row, node = R / p.group;
        QT* o = reinterpret_cast<QT*>(p.out) + (u.s.q0 + node) * p.o_st +
                (int64_t)(u.kvh * p.group + R - node * p.group) * p.o_sh;
        const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (lane + 32 * i < D) o[lane + 32 * i] = from_f32<QT>(acc[r][i] * inv);
      } else {
        float* a = p.part_acc + ((int64_t)slot * kGRows + row) * D;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (lane + 32 * i < D) a[lane + 32 * i] = acc[r][i];
        if (lane == 0)
          p.part_ml[(int64_t)slot * kGRows + row] = make_float2(m[r], l[r] == 0.0f && any[r] ? kSeenInf : l[r]);
      }
    }
  }
}

// ============================================================ combine
// Rows of no sequence (before row `first` and from row `last` on) become 0: threads tid of n, a warp
// per row and head.
template <typename QT>
__device__ __noinline__ void zero_rows(const Params& p, int64_t first, int64_t last, int64_t tid, int64_t n) {
  const int64_t rows = first + p.total_q - last;
  const int lane = tid & 31;
  for (int64_t i = tid >> 5; i < rows * p.num_heads; i += n >> 5) {
    int64_t r = i / p.num_heads;
    const int64_t h = i - r * p.num_heads;
    if (r >= first) r += last - first;
    QT* o = reinterpret_cast<QT*>(p.out) + r * p.o_st + h * p.o_sh;
    for (int d = lane; d < p.head_dim; d += 32) o[d] = from_f32<QT>(0.0f);
  }
}

template <typename QT>
__global__ void __launch_bounds__(128) paged_tree_zero_kernel(const __grid_constant__ Params p) {
  zero_rows<QT>(p, 0, 0, (int64_t)blockIdx.x * 128 + threadIdx.x, (int64_t)gridDim.x * 128);
}

// Joins the parts of each split unit: sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i. CTA
// (c, y) takes rows kCWarps y .. of the unit that desc[c] names, a warp per row: the lanes
// read the parts' maxima and sums side by side, then the parts' rows in order. Four dependent loads
// deep; 4 us behind a small call, 8 us for the 12 MB of parts of a full one. The rows of no sequence
// are this kernel's too where they are to be 0 (their number is known on the device alone).
constexpr int kCWarps = 4;

template <typename QT>
__global__ void __launch_bounds__(32 * kCWarps) paged_tree_combine_kernel(const __grid_constant__ Params p, int RT) {
  int64_t first = 0, last = p.total_q;  // rows of sequences
  if (p.zero_rest) {
    first = ld_idx(p.cu, p.cu_i64, 0);
    last = ld_idx(p.cu, p.cu_i64, p.num_seqs);
  }
  pdl_wait();
  const int4 d = p.desc[2 * blockIdx.x], e = p.desc[2 * blockIdx.x + 1];
  if (first > 0 || last < p.total_q) {
    first = min(max(first, (int64_t)0), p.total_q);
    last = max(min(last, p.total_q), first);
    zero_rows<QT>(p, first, last, ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (32 * kCWarps) + threadIdx.x,
                  (int64_t)gridDim.y * gridDim.x * (32 * kCWarps));
  }
  const int parts_all = d.x, kvh = d.y;
  const int lane = threadIdx.x & 31, row = blockIdx.y * kCWarps + (threadIdx.x >> 5);
  const int R = d.z + row;
  if (parts_all == 0 || row >= RT || R >= d.w) return;
  const int c = blockIdx.x, D = p.head_dim;
  auto slot = [&](int i) -> int64_t { return i == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + i); };
  float M = -INFINITY;
  for (int i = lane; i < parts_all; i += 32) M = fmaxf(M, p.part_ml[slot(i) * RT + row].x);
  M = warp_max(M);
  const float base = M == -INFINITY ? 0.0f : M;
  float L = 0.0f, acc[8];
  bool seen = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  for (int i0 = 0; i0 < parts_all; i0 += 32) {
    float wt = 0.0f, wl = 0.0f;
    if (i0 + lane < parts_all) {  // a part without a visible token has m = -inf and l = 0
      const float2 ml = p.part_ml[slot(i0 + lane) * RT + row];
      wt = exp2f(ml.x - base);
      wl = ml.y == kSeenInf ? 0.0f : wt * ml.y;
      seen |= ml.y == kSeenInf;
    }
    L += warp_sum(wl);
    const int parts = min(32, parts_all - i0);
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float wi = __shfl_sync(0xffffffffu, wt, i);
      const float* a = p.part_acc + (slot(i0 + i) * RT + row) * D;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < D) acc[j] = fmaf(wi, a[lane + 32 * j], acc[j]);
    }
  }
  if (__any_sync(0xffffffffu, seen) && M == -INFINITY) L = NAN;
  const int node = R / p.group;
  const int64_t q0 = ((int64_t)e.x << 32) | (uint32_t)e.y;
  QT* o = reinterpret_cast<QT*>(p.out) + (q0 + node) * p.o_st +
          (int64_t)(kvh * p.group + R - node * p.group) * p.o_sh;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (lane + 32 * j < D) o[lane + 32 * j] = from_f32<QT>(acc[j] * inv);
}

template <typename QT>
int launch_combine(const Params& p, int ctas, int rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int64_t most = p.total_q * p.group;  // rows that a unit can have
  cfg.gridDim = dim3(ctas, ceil_div(most < rows ? most : rows, kCWarps));
  cfg.blockDim = dim3(32 * kCWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, paged_tree_combine_kernel<QT>, p, rows), "paged_tree_combine launch");
}

int launch_zero(const Params& p, int q_dtype, cudaStream_t s) {
  const int64_t warps = p.total_q * p.num_heads, ctas = (warps + 3) / 4, most = 8 * kNumSMs;
  const int grid = (int)(ctas < most ? ctas : most);
  if (q_dtype == MKV_DTYPE_F16) paged_tree_zero_kernel<f16><<<grid, 128, 0, s>>>(p);
  else if (q_dtype == MKV_DTYPE_BF16) paged_tree_zero_kernel<bf16><<<grid, 128, 0, s>>>(p);
  else paged_tree_zero_kernel<float><<<grid, 128, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "paged_tree_zero launch");
}

template <typename QT, typename CT>
int launch_generic(const Params& p, cudaStream_t s) {
  const int bytes = (kGRows * p.head_dim + kGKT * (2 * p.head_dim + 4) + kGRows * kGKT + kGKT) * 4;
  const void* f = (const void*)paged_tree_generic_kernel<QT, CT>;
  int st = ensure_dynamic_smem(f, bytes, "paged_tree_generic shared memory");
  if (st != MKV_OK) return st;
  paged_tree_generic_kernel<QT, CT><<<kGCtas, kGThreads, bytes, s>>>(p);
  return cuda_status(cudaGetLastError(), "paged_tree_generic launch");
}

// How a call is run: the kernel, its row tile and its CTAs.
struct Plan {
  bool tc;
  int rows, ctas;
};

template <typename QT>
int run(const Params& p, const Plan& plan, int q_dtype, int cache_dtype, cudaStream_t s) {
  int st;
  if (plan.tc) st = launch_tc(p, q_dtype, cache_dtype, plan.ctas, s);
  else if (cache_dtype == MKV_DTYPE_FP8_E4M3) st = launch_generic<QT, fp8>(p, s);
  else if (cache_dtype == MKV_DTYPE_INT8) st = launch_generic<QT, int8_t>(p, s);
  else st = launch_generic<QT, QT>(p, s);
  return st == MKV_OK ? launch_combine<QT>(p, plan.ctas, plan.rows, s) : st;
}

std::atomic<int64_t> g_wait_limit{sm100::kWaitCycles};
}  // namespace

int64_t wait_limit() { return g_wait_limit.load(std::memory_order_relaxed); }

Workspace workspace(int ctas, int rows, int head_dim) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  Workspace w;
  w.acc = 0;
  w.ml = up((size_t)2 * ctas * rows * head_dim * 4);
  w.desc = w.ml + up((size_t)2 * ctas * rows * 8);
  w.total = w.desc + up((size_t)ctas * 32);
  return w;
}

}  // namespace tree
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_paged_tree_workspace_bytes(int32_t num_seqs, int64_t total_q, int32_t num_heads,
                                                 int32_t num_kv_heads, int32_t head_dim, int32_t q_dtype,
                                                 int32_t cache_dtype) {
  if (num_seqs <= 0 || total_q <= 0 || num_kv_heads <= 0 || num_heads <= 0 || head_dim <= 0) return 0;
  // the larger of the two kernels' (which of them runs depends on the tensors' alignment too)
  const size_t generic = tree::workspace(tree::kGCtas, tree::kGRows, head_dim).total;
  const size_t tc = tree::workspace(kNumSMs, tree::kTcRows, head_dim).total;
  return (head_dim == 128 || head_dim == 64) && q_dtype != MKV_DTYPE_F32 && tc > generic ? tc : generic;
}

extern "C" int64_t mkv_set_wait_limit(int64_t clocks) {
  return tree::g_wait_limit.exchange(clocks < 0 ? 0 : clocks, std::memory_order_relaxed);
}

#define TREE_PARAMETERS \
    const void* query, int64_t q_stride_token, int64_t q_stride_head, int32_t q_dtype, \
    const void* k_cache, const void* v_cache, int32_t cache_dtype, const float* k_scale, \
    const float* v_scale, const float* k_scales, const float* v_scales, int64_t num_blocks, \
    int32_t block_size, const void* block_tables, int32_t block_table_index_type, \
    int64_t block_table_stride_seq, int32_t max_num_blocks, const void* context_lens, \
    int32_t context_lens_index_type, const void* cu_seqlens_q, int32_t cu_seqlens_index_type, \
    const uint64_t* tree_mask, int64_t mask_stride_token, int32_t mask_words, int32_t num_seqs, \
    int64_t total_q, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale, \
    void* out, int64_t out_stride_token, int64_t out_stride_head, void* workspace, \
    size_t workspace_bytes, void* stream
#define TREE_ARGUMENTS \
    query, q_stride_token, q_stride_head, q_dtype, k_cache, v_cache, cache_dtype, k_scale, v_scale, k_scales, \
    v_scales, num_blocks, block_size, block_tables, block_table_index_type, block_table_stride_seq, \
    max_num_blocks, context_lens, context_lens_index_type, cu_seqlens_q, cu_seqlens_index_type, tree_mask, \
    mask_stride_token, mask_words, num_seqs, total_q, num_heads, num_kv_heads, head_dim, scale, out, \
    out_stride_token, out_stride_head, workspace, workspace_bytes, stream

namespace {
int tree_attention(const char* fn, bool zero_rest, TREE_PARAMETERS) {
  clear_error();
  if (num_seqs < 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      max_num_blocks < 0 || num_blocks < 0 || mask_words < 1)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: bad sizes", fn);
  if (num_heads % num_kv_heads != 0)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: num_heads must be a multiple of num_kv_heads", fn);
  if (head_dim % 16 != 0 || head_dim > 256)
    return set_error(MKV_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16, at most 256 (got %d)", fn, head_dim);
  // (token indices are 32-bit, and are formed for the three tiles of 128 behind a context's last one too)
  if ((int64_t)max_num_blocks * block_size > 0x7fffffffll - 1023)
    return set_error(MKV_ERR_UNSUPPORTED, "%s: max_num_blocks x block_size exceeds 2^31 tokens (less 1024)", fn);
  if (total_q > 0x7fffffffll / (num_heads / num_kv_heads))
    return set_error(MKV_ERR_UNSUPPORTED, "%s: total_q x query heads per kv head exceeds 2^31", fn);
  if (q_dtype != MKV_DTYPE_F32 && q_dtype != MKV_DTYPE_F16 && q_dtype != MKV_DTYPE_BF16)
    return set_error(MKV_ERR_UNSUPPORTED, "%s: query dtype must be f32, f16 or bf16", fn);
  for (int32_t t : {block_table_index_type, context_lens_index_type, cu_seqlens_index_type})
    if (t != MKV_INDEX_I32 && t != MKV_INDEX_I64)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: index types must be MKV_INDEX_I32 or MKV_INDEX_I64", fn);
  const bool byte = cache_dtype == MKV_DTYPE_FP8_E4M3 || cache_dtype == MKV_DTYPE_INT8;
  const bool tensor_scales = k_scale || v_scale, row_scales = k_scales || v_scales;
  if (!byte && cache_dtype != q_dtype)
    return set_error(MKV_ERR_UNSUPPORTED, "%s: the cache dtype must be the query's, FP8_E4M3 or INT8", fn);
  if (!byte && (tensor_scales || row_scales))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: scales given for an unquantised cache", fn);
  if (byte && (tensor_scales == row_scales || (tensor_scales && (!k_scale || !v_scale)) ||
               (row_scales && (!k_scales || !v_scales))))
    return set_error(MKV_ERR_INVALID_ARGUMENT,
                     "%s: an 8-bit cache needs k_scale and v_scale, or k_scales and v_scales", fn);
  if (cache_dtype == MKV_DTYPE_INT8 && !row_scales)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: an INT8 cache needs k_scales and v_scales", fn);
  if (total_q == 0 || (num_seqs == 0 && !zero_rest)) return MKV_OK;
  if (num_seqs > 0 && (!query || !tree_mask || !context_lens || !cu_seqlens_q ||
                       (max_num_blocks > 0 && !block_tables) || (num_blocks > 0 && (!k_cache || !v_cache))))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (!out) return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: caches must be 16-byte aligned", fn);
  const size_t need = mkv_paged_tree_workspace_bytes(num_seqs, total_q, num_heads, num_kv_heads, head_dim, q_dtype,
                                                     cache_dtype);
  if (num_seqs > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return set_error(MKV_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", fn, need,
                     workspace ? workspace_bytes : (size_t)0);
  tree::Params p = {};
  p.q = query;
  p.q_st = q_stride_token;
  p.q_sh = q_stride_head;
  p.k_cache = (const uint8_t*)k_cache;
  p.v_cache = (const uint8_t*)v_cache;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.bt = block_tables;
  p.bt_sb = block_table_stride_seq;
  p.max_blocks = max_num_blocks;
  p.bt_i64 = block_table_index_type == MKV_INDEX_I64;
  p.ctx = context_lens;
  p.ctx_i64 = context_lens_index_type == MKV_INDEX_I64;
  p.cu = cu_seqlens_q;
  p.cu_i64 = cu_seqlens_index_type == MKV_INDEX_I64;
  p.mask = tree_mask;
  p.mask_st = mask_stride_token;
  p.mask_words = mask_words;
  p.num_seqs = num_seqs;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.group = num_heads / num_kv_heads;
  p.total_q = total_q;
  p.qk_scale_log2 = scale * 1.4426950408889634f;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.out = out;
  p.o_st = out_stride_token;
  p.o_sh = out_stride_head;
  p.zero_rest = zero_rest;
  p.wait_limit = tree::wait_limit();
  cudaStream_t s = (cudaStream_t)stream;
  if (num_seqs == 0) return tree::launch_zero(p, q_dtype, s);
  const tree::Plan plan = tree::tc_supported(p, q_dtype, cache_dtype)
                              ? tree::Plan{true, tree::kTcRows, kNumSMs}
                              : tree::Plan{false, tree::kGRows, tree::kGCtas};
  p.unit_cost = plan.tc ? (cache_dtype == q_dtype ? 4 : 2) : 0;
  const tree::Workspace w = tree::workspace(plan.ctas, plan.rows, head_dim);
  p.part_acc = (float*)((char*)workspace + w.acc);
  p.part_ml = (float2*)((char*)workspace + w.ml);
  p.desc = (int4*)((char*)workspace + w.desc);
  switch (q_dtype) {
    case MKV_DTYPE_F16: return tree::run<f16>(p, plan, q_dtype, cache_dtype, s);
    case MKV_DTYPE_BF16: return tree::run<bf16>(p, plan, q_dtype, cache_dtype, s);
    default: return tree::run<float>(p, plan, q_dtype, cache_dtype, s);
  }
}
}  // namespace

extern "C" int mkv_paged_tree_attention(TREE_PARAMETERS) {
  return tree_attention("mkv_paged_tree_attention", false, TREE_ARGUMENTS);
}
extern "C" int mkv_paged_tree_attention_zeroed(TREE_PARAMETERS) {
  return tree_attention("mkv_paged_tree_attention_zeroed", true, TREE_ARGUMENTS);
}
