// Metadata and verification of a decode step over trees of drafted tokens.
//
// Sequence b of the step has prefix[b] cached tokens and n_b drafted nodes, rows
// [cu[b], cu[b + 1]) of the step's arrays, node 0 the tree's root. parents[row] is the
// node's parent within its own tree (a lower index), -1 for a root.
//
// mkv_tree_metadata: node i of sequence b is cached at position prefix + i and sits at
// sequence position prefix + depth(i); it attends to itself and its ancestors, one bit
// each in the mask row.
// mkv_tree_accept: the path that the target model agrees with. It starts at node 0; after
// node c comes its lowest child d with draft[d] == target[c]; target[c] is the token that
// follows c, so the path's targets are the step's new tokens, the last one not drafted.
//
// Both are bound by launch and load latency (a batch of 256 trees of 64 nodes holds half a
// megabyte), so each is one launch, with a chain of dependent loads that does not grow
// with the number of nodes: a tree is read once, into shared memory or registers, and
// walked there. Measured (B200, graph replays): metadata of 1 / 256 trees 2.8 / 3.4 us,
// acceptance 3.1 / 5.1 us, about what an empty launch takes.
#include "mkv_common.cuh"

namespace mkv {
namespace {

__device__ __forceinline__ int64_t ts_index(const void* p, int i64, int64_t i) {
  return i64 ? __ldg(reinterpret_cast<const int64_t*>(p) + i)
             : (int64_t)__ldg(reinterpret_cast<const int32_t*>(p) + i);
}

struct TreeParams {
  const void* parents;
  const void* cu;
  const void* prefix;
  const void* bt;
  int64_t bt_stride;
  int parents_i64, cu_i64, prefix_i64, bt_i64;
  int max_blocks, block_size, num_seqs;
  int64_t total_q;
};

// First row and number of nodes of sequence b, within [0, total_q).
__device__ __forceinline__ void ts_rows(const TreeParams& p, int b, int64_t& q0, int64_t& n) {
  q0 = ts_index(p.cu, p.cu_i64, b);
  int64_t q1 = ts_index(p.cu, p.cu_i64, b + 1);
  q0 = min(max(q0, (int64_t)0), p.total_q);
  q1 = min(max(q1, (int64_t)0), p.total_q);
  n = max(q1 - q0, (int64_t)0);
}

__device__ __forceinline__ int64_t ts_prefix(const TreeParams& p, int b) {
  return max(ts_index(p.prefix, p.prefix_i64, b), (int64_t)0);
}

// Cache slot of token `j` behind the prefix of sequence b, -1 where it has no page.
__device__ __forceinline__ int64_t ts_slot(const TreeParams& p, int b, int64_t prefix, int64_t j) {
  if (prefix >= (int64_t)p.max_blocks * p.block_size - j) return -1;  // (the sum may pass 64 bits)
  const int64_t pos = prefix + j, blk = pos / p.block_size;
  const int64_t page = ts_index(p.bt, p.bt_i64, b * p.bt_stride + blk);
  return page < 0 ? -1 : page * p.block_size + (pos - blk * p.block_size);
}

constexpr int kMetaThreads = 128;
constexpr int kMaxWords = 16;  // 1024 nodes a tree

// One CTA per sequence, and a last one for the rows that belong to none (a captured
// step's padding), whose slots are -1 so that the append skips them. Parents are staged in
// shared memory; a thread walks its node's chain up to the root. Ancestors have lower
// indices, so the words of the mask row are completed from the highest down.
__global__ void __launch_bounds__(kMetaThreads)
tree_metadata_kernel(const TreeParams p, int words, int64_t* slots, int64_t* lens,
                     int64_t* positions, uint64_t* mask, int32_t* invalid_count) {
  __shared__ int par[64 * kMaxWords];
  const int b = blockIdx.x, tid = threadIdx.x;
  if (b == p.num_seqs) {
    const int64_t first = min(max(ts_index(p.cu, p.cu_i64, 0), (int64_t)0), p.total_q);
    const int64_t last = min(max(ts_index(p.cu, p.cu_i64, p.num_seqs), (int64_t)0), p.total_q);
    const int64_t behind = max(last, first);
    for (int64_t i = tid; i < first + (p.total_q - behind); i += kMetaThreads) {
      const int64_t r = i < first ? i : behind + (i - first);
      slots[r] = -1;
      positions[r] = 0;
      for (int w = 0; w < words; ++w) mask[r * words + w] = 0;
    }
    return;
  }
  int64_t q0, n64;
  ts_rows(p, b, q0, n64);
  const int64_t prefix = ts_prefix(p, b);
  const int cap = 64 * words;
  const int n = n64 < cap ? (int)n64 : cap;  // nodes that the mask can name
  int bad = 0;
  for (int j = tid; j < n; j += kMetaThreads) {
    const int64_t v = ts_index(p.parents, p.parents_i64, q0 + j);
    const bool ok = v >= -1 && v < j;
    par[j] = ok ? (int)v : -1;
    bad += !ok;
  }
  __syncthreads();
  for (int j = tid; j < n; j += kMetaThreads) {
    uint64_t* row = mask + (q0 + j) * words;
    int w = j >> 6, depth = 0;
    for (int x = words - 1; x > w; --x) row[x] = 0;
    uint64_t acc = 1ull << (j & 63);
    for (int a = par[j]; a >= 0; a = par[a]) {  // a falls at every step: at most j of them
      ++depth;
      for (const int wa = a >> 6; w > wa; acc = 0) row[w--] = acc;
      acc |= 1ull << (a & 63);
    }
    for (; w >= 0; acc = 0) row[w--] = acc;
    slots[q0 + j] = ts_slot(p, b, prefix, j);
    positions[q0 + j] = prefix + depth;
  }
  for (int64_t j = n + tid; j < n64; j += kMetaThreads) {  // past the mask's width: not cached, sees nothing
    slots[q0 + j] = -1;
    positions[q0 + j] = prefix;
    for (int w = 0; w < words; ++w) mask[(q0 + j) * words + w] = 0;
    ++bad;
  }
  if (tid == 0) lens[b] = prefix + n64;
  if (invalid_count != nullptr && bad) atomicAdd(invalid_count, bad);
}

constexpr int kAcceptWarps = 4;
constexpr int kHeld = 4;  // nodes a lane holds in registers: trees of up to 128 nodes

// One warp per sequence. Lane l holds nodes l, l + 32, ...: a step of the path is a
// comparison of the held nodes and a ballot, with no load; nodes past the held ones are
// read from memory.
__global__ void __launch_bounds__(32 * kAcceptWarps)
tree_accept_kernel(const TreeParams p, const void* draft, const void* target, int tok_i64,
                   int max_path, int32_t* num_accepted, int32_t* accepted, int64_t* tokens,
                   int64_t* lens, int64_t* src, int64_t* dst) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.x * kAcceptWarps + (threadIdx.x >> 5);
  if (b >= p.num_seqs) return;
  int64_t q0, n;
  ts_rows(p, b, q0, n);
  const int64_t prefix = ts_prefix(p, b);
  int64_t hp[kHeld], hd[kHeld], ht[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int64_t j = lane + 32 * i;
    const bool in = j < n;
    hp[i] = in ? ts_index(p.parents, p.parents_i64, q0 + j) : -1;
    hd[i] = in ? ts_index(draft, tok_i64, q0 + j) : 0;
    ht[i] = in ? ts_index(target, tok_i64, q0 + j) : 0;
  }
  int64_t cur = n > 0 ? 0 : -1;
  int count = 0;
  int64_t* row_t = tokens + (int64_t)b * max_path;
  int32_t* row_n = accepted + (int64_t)b * max_path;
  // the step's path is collected 32 entries at a time, lane k % 32 holding entry k
  int64_t my_node = -1, my_tok = -1;
  int k = 0;
  auto flush = [&](int base) {
    const int e = base + lane;
    if (e >= max_path) return;
    row_n[e] = (int32_t)my_node;
    row_t[e] = my_tok;
    const bool moved = my_node >= 0 && my_node != e;
    src[(int64_t)b * max_path + e] = moved ? ts_slot(p, b, prefix, my_node) : -1;
    dst[(int64_t)b * max_path + e] = moved ? ts_slot(p, b, prefix, e) : -1;
    my_node = my_tok = -1;
  };
  for (k = 0; k < max_path; ++k) {
    if (cur >= 0) {
      int64_t tok = 0;
      if (cur < 32 * kHeld) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          const int64_t v = __shfl_sync(0xffffffffu, ht[i], (int)(cur & 31));
          if ((cur >> 5) == i) tok = v;
        }
      } else {
        tok = ts_index(target, tok_i64, q0 + cur);
      }
      if (lane == (k & 31)) {
        my_node = cur;
        my_tok = tok;
      }
      ++count;
      int64_t next = -1;
#pragma unroll
      for (int i = kHeld - 1; i >= 0; --i) {
        const int64_t j = lane + 32 * i;
        const unsigned m = __ballot_sync(0xffffffffu, j < n && j > cur && hp[i] == cur && hd[i] == tok);
        if (m) next = 32 * i + __ffs(m) - 1;
      }
      for (int64_t base = 32 * kHeld; next < 0 && base < n; base += 32) {
        const int64_t j = base + lane;
        const bool fits = j < n && j > cur && ts_index(p.parents, p.parents_i64, q0 + j) == cur &&
                          ts_index(draft, tok_i64, q0 + j) == tok;
        const unsigned m = __ballot_sync(0xffffffffu, fits);
        if (m) next = base + __ffs(m) - 1;
      }
      cur = next;
    }
    if ((k & 31) == 31) flush(k - 31);
  }
  if (k & 31) flush(k & ~31);
  if (lane == 0) {
    num_accepted[b] = count;
    lens[b] = prefix + count;
  }
}

int check_tree(const char* fn, const void* parents, int32_t parents_type, const void* cu, int32_t cu_type,
               const void* prefix, int32_t prefix_type, const void* bt, int32_t bt_type,
               int32_t max_blocks, int32_t block_size, int32_t num_seqs, int64_t total_q) {
  if (num_seqs < 0 || total_q < 0 || max_blocks < 0 || block_size <= 0)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: bad sizes", fn);
  for (int32_t t : {parents_type, cu_type, prefix_type, bt_type})
    if (t != MKV_INDEX_I32 && t != MKV_INDEX_I64)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: index types must be MKV_INDEX_I32 or MKV_INDEX_I64", fn);
  if (num_seqs > 0 && ((total_q > 0 && !parents) || !cu || !prefix || (max_blocks > 0 && !bt)))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  return MKV_OK;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int mkv_tree_metadata(const void* parents, int32_t parents_index_type, const void* cu_seqlens_q,
                                 int32_t cu_seqlens_index_type, const void* prefix_lens,
                                 int32_t prefix_lens_index_type, const void* block_tables,
                                 int32_t block_table_index_type, int64_t block_table_stride_seq,
                                 int32_t max_num_blocks, int32_t block_size, int32_t num_seqs,
                                 int64_t total_q, int32_t mask_words, int64_t* slot_mapping,
                                 int64_t* context_lens, int64_t* positions, uint64_t* tree_mask,
                                 int32_t* invalid_count, void* stream) {
  clear_error();
  const char* fn = "mkv_tree_metadata";
  const int st = check_tree(fn, parents, parents_index_type, cu_seqlens_q, cu_seqlens_index_type, prefix_lens,
                            prefix_lens_index_type, block_tables, block_table_index_type, max_num_blocks,
                            block_size, num_seqs, total_q);
  if (st != MKV_OK) return st;
  if (mask_words < 1 || mask_words > kMaxWords)
    return set_error(MKV_ERR_UNSUPPORTED, "%s: mask_words must be 1 to %d (got %d)", fn, kMaxWords, mask_words);
  if (num_seqs == 0 && total_q == 0) return MKV_OK;
  if (!cu_seqlens_q) return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if ((num_seqs > 0 && !context_lens) || (total_q > 0 && (!slot_mapping || !positions || !tree_mask)))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null output pointer", fn);
  TreeParams p{parents, cu_seqlens_q, prefix_lens, block_tables, block_table_stride_seq,
               parents_index_type == MKV_INDEX_I64, cu_seqlens_index_type == MKV_INDEX_I64,
               prefix_lens_index_type == MKV_INDEX_I64, block_table_index_type == MKV_INDEX_I64,
               max_num_blocks, block_size, num_seqs, total_q};
  tree_metadata_kernel<<<num_seqs + 1, kMetaThreads, 0, (cudaStream_t)stream>>>(
      p, mask_words, slot_mapping, context_lens, positions, tree_mask, invalid_count);
  return cuda_status(cudaGetLastError(), "tree_metadata launch");
}

extern "C" int mkv_tree_accept(const void* draft_tokens, const void* target_tokens, int32_t token_index_type,
                               const void* parents, int32_t parents_index_type, const void* cu_seqlens_q,
                               int32_t cu_seqlens_index_type, const void* prefix_lens,
                               int32_t prefix_lens_index_type, const void* block_tables,
                               int32_t block_table_index_type, int64_t block_table_stride_seq,
                               int32_t max_num_blocks, int32_t block_size, int32_t num_seqs, int64_t total_q,
                               int32_t max_path, int32_t* num_accepted, int32_t* accepted_nodes,
                               int64_t* tokens, int64_t* context_lens, int64_t* src_slots, int64_t* dst_slots,
                               void* stream) {
  clear_error();
  const char* fn = "mkv_tree_accept";
  const int st = check_tree(fn, parents, parents_index_type, cu_seqlens_q, cu_seqlens_index_type, prefix_lens,
                            prefix_lens_index_type, block_tables, block_table_index_type, max_num_blocks,
                            block_size, num_seqs, total_q);
  if (st != MKV_OK) return st;
  if (token_index_type != MKV_INDEX_I32 && token_index_type != MKV_INDEX_I64)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: token_index_type must be MKV_INDEX_I32 or MKV_INDEX_I64", fn);
  if (max_path < 1) return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: max_path must be at least 1", fn);
  if (num_seqs == 0) return MKV_OK;
  if ((total_q > 0 && (!draft_tokens || !target_tokens)) || !num_accepted || !accepted_nodes || !tokens ||
      !context_lens || !src_slots || !dst_slots)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  TreeParams p{parents, cu_seqlens_q, prefix_lens, block_tables, block_table_stride_seq,
               parents_index_type == MKV_INDEX_I64, cu_seqlens_index_type == MKV_INDEX_I64,
               prefix_lens_index_type == MKV_INDEX_I64, block_table_index_type == MKV_INDEX_I64,
               max_num_blocks, block_size, num_seqs, total_q};
  tree_accept_kernel<<<ceil_div(num_seqs, kAcceptWarps), 32 * kAcceptWarps, 0, (cudaStream_t)stream>>>(
      p, draft_tokens, target_tokens, token_index_type == MKV_INDEX_I64, max_path, num_accepted,
      accepted_nodes, tokens, context_lens, src_slots, dst_slots);
  return cuda_status(cudaGetLastError(), "tree_accept launch");
}
