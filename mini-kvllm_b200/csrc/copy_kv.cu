// Copies of cached data inside the paged KV cache, over every layer, K and V and the row
// scales in one launch (several, one for each 1024 pairs, where the pairs are split): whole pages (a
// fork's private copy of a shared page, compaction of a fragmented cache) and single rows (the accepted rows of a tree of drafted tokens,
// moved to the end of the cached prefix).
//
// A copy moves `unit` bytes (a page, or one token's row of all kv heads) from unit src[i]
// to unit dst[i] of every plane (layer x {K, V}, and their scales). Copies are applied in
// order i = 0, 1, ..., each seeing what the earlier ones wrote, whatever the indices
// repeat: a thread owns a 16-byte column of the unit in a few layers and makes all copies of
// its columns itself, so no other thread ever touches those bytes and program order is the
// only order needed. Four copies of two layers are in flight per thread (loads first, then
// stores); when a copy of the four reads what an earlier one of them writes, they are made one
// at a time.
//
// Bound: memory, 2 x unit bytes a copy. The columns of a whole cache (28 layers of 32 KB
// pages: 114688, two layers to a thread) keep 57344 threads x 128 bytes = 7.3 MB in flight, enough
// to cover the latency of HBM, and the threads fit the GPU at once (233 pairs: 140 us, 6.1 TB/s, 0.94
// of the copy rate; three pairs 3.4 us).
// Where the columns are few and the pairs many (small pages of one kv head), the pairs are split
// over CTAs as well, if none of them writes what another one reads or writes: every CTA finds
// that out for itself, with a hash table of the destinations.
// A group of row copies is one sequence's, groups side by side; there a
// thread's layers share the reading and checking of the indices.
#include "mkv_common.cuh"

namespace mkv {
namespace {

constexpr int kCopyThreads = 128;
constexpr int kInFlight = 4;
constexpr int kCopyCtas = 5;  // resident on an SM
constexpr int kSplitPairs = 1024, kHashSlots = 2 * kSplitPairs;  // pairs of a launch that may split them

struct CopyParams {
  uint8_t* base[2];      // K and V of layer 0
  uint8_t* sbase[2];     // their row scales, or null
  int64_t plane_stride;  // bytes from layer to layer
  int64_t splane_stride;
  int64_t unit;          // bytes of a unit of K or V
  int64_t sunit;         // and of its scales (0: none)
  int svec;              // column width of the scales, 16 or 4 bytes (K and V: 16)
  int64_t num_units;
  int num_layers;
  int per_thread;        // layers that a thread takes
  const void* src;
  const void* dst;
  int i64;
  int num_copies;        // of a group
  int num_groups;
  int32_t* invalid_count;
};

__device__ __forceinline__ int64_t cp_index(const CopyParams& c, const void* p, int64_t i) {
  return c.i64 ? __ldg(reinterpret_cast<const int64_t*>(p) + i)
               : (int64_t)__ldg(reinterpret_cast<const int32_t*>(p) + i);
}

// Loads and stores where `on`, in program order (volatile, with a memory clobber): a thread
// may read what it has written. Predicated, not branched around: the loads of a batch stay
// together.
__device__ __forceinline__ void cp_load(const uint8_t* p, bool on, uint4& r) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
      : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
      : "l"(p), "r"((int)on)
      : "memory");
}
__device__ __forceinline__ void cp_load(const uint8_t* p, bool on, uint32_t& r) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.u32 %0, [%1];\n\t}"
               : "+r"(r)
               : "l"(p), "r"((int)on)
               : "memory");
}
__device__ __forceinline__ void cp_store(uint8_t* p, bool on, const uint4& v) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q st.global.v4.u32 [%0], {%1,%2,%3,%4};\n\t}" ::"l"(p),
      "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"((int)on)
      : "memory");
}
__device__ __forceinline__ void cp_store(uint8_t* p, bool on, uint32_t v) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q st.global.u32 [%0], %1;\n\t}" ::"l"(p), "r"(v),
               "r"((int)on)
               : "memory");
}

// All copies of one column of a group in `layers` layers, `stride` bytes apart: p points at its
// bytes in unit 0 of the first, T is its type. A negative entry is no copy; one past the cache
// is skipped. A unit's copy onto itself is left out: done as a load and a store it would put old
// bytes over those that another CTA, with another part of the pairs, has copied there.
template <typename T>
__device__ __forceinline__ void copy_column(const CopyParams& c, uint8_t* p, int64_t stride, int layers,
                                            int64_t unit, int64_t first, int count) {
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += kInFlight) {
    int64_t s[kInFlight], d[kInFlight];
    bool chained = false, any = false;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      s[u] = d[u] = -1;
      if (i0 + u < count) {
        s[u] = cp_index(c, c.src, first + i0 + u);
        d[u] = cp_index(c, c.dst, first + i0 + u);
      }
      if (s[u] < 0 || d[u] < 0 || s[u] >= c.num_units || d[u] >= c.num_units || s[u] == d[u]) s[u] = d[u] = -1;
      any |= s[u] >= 0;
#pragma unroll
      for (int w = 0; w < u; ++w) chained |= s[u] >= 0 && s[u] == d[w];
    }
    if (!any) continue;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {  // byte offsets from here on
      if (s[u] >= 0) {
        s[u] *= unit;
        d[u] *= unit;
      }
    }
    uint8_t* q = p;
    if (!chained) {
#pragma unroll 1
      for (int l = 0; l < layers; l += 2, q += 2 * stride) {
        const bool two = l + 1 < layers;
        T x[2][kInFlight] = {};
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
          cp_load(q + s[u], s[u] >= 0, x[0][u]);
          cp_load(q + stride + s[u], s[u] >= 0 && two, x[1][u]);
        }
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
          cp_store(q + d[u], s[u] >= 0, x[0][u]);
          cp_store(q + stride + d[u], s[u] >= 0 && two, x[1][u]);
        }
      }
    } else {
#pragma unroll 1
      for (int l = 0; l < layers; ++l, q += stride) {
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
          T x = {};
          cp_load(q + s[u], s[u] >= 0, x);
          cp_store(q + d[u], s[u] >= 0, x);
        }
      }
    }
  }
}

// Whether some pair of c writes a unit that another one reads or writes (copies of a unit onto
// itself read and write nothing). Block-collective; the same answer in every block.
__device__ bool pairs_clash(const CopyParams& c) {
  __shared__ long long table[kHashSlots];
  __shared__ int clash;
  for (int i = threadIdx.x; i < kHashSlots; i += kCopyThreads) table[i] = -1;
  if (threadIdx.x == 0) clash = 0;
  __syncthreads();
  auto slot = [](int64_t v) { return (uint32_t)((uint64_t)v * 0x9E3779B97F4A7C15ull >> 53); };  // 11 bits
  static_assert(kHashSlots == 2048, "slot() has 11 bits");
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // enter the destinations, then look the sources up
#pragma unroll 1
    for (int i = threadIdx.x; i < c.num_copies; i += kCopyThreads) {
      const int64_t s = cp_index(c, c.src, i), d = cp_index(c, c.dst, i);
      if (s < 0 || d < 0 || s >= c.num_units || d >= c.num_units || s == d) continue;
      uint32_t h = slot(pass ? s : d);
      while (true) {  // at most half of the slots are taken: it ends
        const long long old = pass ? table[h]
                                   : (long long)atomicCAS((unsigned long long*)&table[h], (unsigned long long)-1ll,
                                                          (unsigned long long)d);
        if (old == -1) break;
        if (old == (pass ? s : d)) {
          clash = 1;
          break;
        }
        h = (h + 1) & (kHashSlots - 1);
      }
    }
    __syncthreads();
  }
  return clash != 0;
}

// kSplit: one group, whose pairs are spread over blockIdx.y where they do not clash.
template <bool kSplit>
__global__ void __launch_bounds__(kCopyThreads, kCopyCtas) copy_units_kernel(const __grid_constant__ CopyParams c) {
  const int64_t cols = c.unit / 16, scols = c.sunit ? c.sunit / c.svec : 0;
  const int64_t parts = (c.num_layers + c.per_thread - 1) / c.per_thread;  // of the layers
  const int64_t at = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  int begin = 0, end = c.num_copies;
  if constexpr (kSplit) {
    const bool whole = pairs_clash(c);
    if (!whole) {
      begin = (int)((int64_t)c.num_copies * blockIdx.y / gridDim.y);
      end = (int)((int64_t)c.num_copies * (blockIdx.y + 1) / gridDim.y);
    } else if (blockIdx.y > 0) {
      return;
    }
  }
  for (int g = kSplit ? 0 : blockIdx.y; g < c.num_groups; g += kSplit ? 1 : gridDim.y) {
    const int64_t first = (int64_t)g * c.num_copies + begin;
    const bool values = at < 2 * parts * cols;
    const int64_t a = values ? at : at - 2 * parts * cols;
    const int64_t n = values ? cols : scols;
    if (n > 0 && a < 2 * parts * n) {
      const int64_t part = a / n, col = a - part * n;
      const int l0 = (int)(part >> 1) * c.per_thread, layers = min(c.per_thread, c.num_layers - l0);
      if (values)
        copy_column<uint4>(c, (part & 1 ? c.base[1] : c.base[0]) + l0 * c.plane_stride + col * 16, c.plane_stride, layers,
                           c.unit, first, end - begin);
      else if (c.svec == 16)
        copy_column<uint4>(c, (part & 1 ? c.sbase[1] : c.sbase[0]) + l0 * c.splane_stride + col * 16, c.splane_stride,
                           layers, c.sunit, first, end - begin);
      else
        copy_column<uint32_t>(c, (part & 1 ? c.sbase[1] : c.sbase[0]) + l0 * c.splane_stride + col * 4, c.splane_stride,
                              layers, c.sunit, first, end - begin);
    }
    if (c.invalid_count != nullptr && blockIdx.x == 0) {
      int bad = 0;
      for (int i = begin + threadIdx.x; i < end; i += kCopyThreads) {
        const int64_t at = (int64_t)g * c.num_copies + i;
        const int64_t s = cp_index(c, c.src, at), d = cp_index(c, c.dst, at);
        bad += s >= 0 && d >= 0 && (s >= c.num_units || d >= c.num_units);
      }
      if (bad) atomicAdd(c.invalid_count, bad);
    }
  }
}

int copy_units(const char* fn, void* k_cache, void* v_cache, int32_t cache_dtype, int32_t num_layers,
               int64_t layer_stride, int64_t num_blocks, int32_t block_size, int32_t num_kv_heads,
               int32_t head_dim, float* k_scales, float* v_scales, int64_t scale_layer_stride,
               const void* src, const void* dst, int32_t index_type, int32_t num_groups,
               int64_t num_copies, bool pages, int32_t* invalid_count, void* stream) {
  if (num_layers < 0 || num_blocks < 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      num_groups < 0 || num_copies < 0 || num_copies > 0x7fffffff - kInFlight)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: bad sizes", fn);
  const int bytes = cache_dtype == MKV_DTYPE_INT8 ? 1 : dtype_bytes(cache_dtype);
  if (bytes == 0) return set_error(MKV_ERR_UNSUPPORTED, "%s: unsupported cache dtype %d", fn, cache_dtype);
  if (index_type != MKV_INDEX_I32 && index_type != MKV_INDEX_I64)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: index_type must be MKV_INDEX_I32 or MKV_INDEX_I64", fn);
  if ((k_scales == nullptr) != (v_scales == nullptr))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: k_scales and v_scales must both be given or both be NULL", fn);
  const int64_t row = (int64_t)num_kv_heads * head_dim * bytes;
  if (row % 16 != 0)
    return set_error(MKV_ERR_UNSUPPORTED, "%s: a token's row of %lld bytes is not a multiple of 16", fn,
                     (long long)row);
  if (num_copies == 0 || num_groups == 0 || num_layers == 0 || num_blocks == 0) return MKV_OK;
  if (!k_cache || !v_cache || !src || !dst)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (((uintptr_t)k_cache | (uintptr_t)v_cache | (uint64_t)(layer_stride * bytes)) & 15)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: caches and layers must be 16-byte aligned", fn);
  if (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: scales must be 4-byte aligned", fn);
  CopyParams c;
  c.base[0] = (uint8_t*)k_cache;
  c.base[1] = (uint8_t*)v_cache;
  c.sbase[0] = (uint8_t*)k_scales;
  c.sbase[1] = (uint8_t*)v_scales;
  c.plane_stride = layer_stride * bytes;
  c.splane_stride = scale_layer_stride * 4;
  const int64_t rows = pages ? block_size : 1;
  c.unit = row * rows;
  c.sunit = k_scales ? rows * num_kv_heads * 4 : 0;
  c.svec = (((uintptr_t)k_scales | (uintptr_t)v_scales | (uint64_t)c.sunit | (uint64_t)c.splane_stride) & 15) ? 4 : 16;
  c.num_units = pages ? num_blocks : num_blocks * block_size;
  c.num_layers = num_layers;
  c.src = src;
  c.dst = dst;
  c.i64 = index_type == MKV_INDEX_I64;
  c.num_copies = (int)num_copies;
  c.num_groups = num_groups;
  c.invalid_count = invalid_count;
  // layers a thread, at most 8: as many as bring the grid down to what is resident at once (a page copy
  // in two waves takes 1.5 times as long), and no more: one stream's move of a few rows is bound by
  // latency and wants a thread for each column, a batch's reads its indices less often this way (44 us
  // against 92 for 253 sequences of up to 7 moves).
  const int64_t unit_cols = c.unit / 16 + (c.sunit ? c.sunit / c.svec : 0);
  const int64_t resident = (int64_t)kNumSMs * kCopyCtas * kCopyThreads;
  const int groups = num_groups < 65535 ? num_groups : 65535;
  const int64_t threads = 2 * unit_cols * num_layers;  // of a group, with a layer each
  const int64_t waves = (threads * groups + resident - 1) / resident;
  c.per_thread = (int)(waves < 1 ? 1 : waves > 8 ? 8 : waves);
  const int64_t columns = 2 * unit_cols * ((num_layers + c.per_thread - 1) / c.per_thread);
  const int64_t ctas = (columns + kCopyThreads - 1) / kCopyThreads;
  if (ctas > 0x7fffffff) return set_error(MKV_ERR_INVALID_ARGUMENT, "%s: bad sizes", fn);
  // Few columns and many pairs (28 layers of 2 KB pages: 7168 threads, a tenth of what fits): the pairs
  // are split, in launches of at most kSplitPairs, until the GPU is full or a CTA has kInFlight of them.
  if (num_groups == 1 && num_copies >= 4 * kInFlight && 2 * threads <= resident) {
    const int isize = c.i64 ? 8 : 4;
    for (int64_t i = 0; i < num_copies; i += kSplitPairs) {
      CopyParams part = c;
      part.num_copies = (int)(num_copies - i < kSplitPairs ? num_copies - i : kSplitPairs);
      part.src = (const uint8_t*)src + i * isize;
      part.dst = (const uint8_t*)dst + i * isize;
      int64_t splits = resident / threads, most = (part.num_copies + kInFlight - 1) / kInFlight;
      if (splits > most) splits = most;
      copy_units_kernel<true><<<dim3((unsigned)ctas, (unsigned)splits), kCopyThreads, 0, (cudaStream_t)stream>>>(part);
      const int st = cuda_status(cudaGetLastError(), "copy_units launch");
      if (st != MKV_OK) return st;
    }
    return MKV_OK;
  }
  copy_units_kernel<false><<<dim3((unsigned)ctas, (unsigned)groups), kCopyThreads, 0, (cudaStream_t)stream>>>(c);
  return cuda_status(cudaGetLastError(), "copy_units launch");
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int mkv_copy_kv_pages(void* k_cache, void* v_cache, int32_t cache_dtype, int32_t num_layers,
                                 int64_t layer_stride, int64_t num_blocks, int32_t block_size,
                                 int32_t num_kv_heads, int32_t head_dim, float* k_scales, float* v_scales,
                                 int64_t scale_layer_stride, const void* src_pages, const void* dst_pages,
                                 int32_t index_type, int64_t num_pairs, int32_t* invalid_count, void* stream) {
  clear_error();
  return copy_units("mkv_copy_kv_pages", k_cache, v_cache, cache_dtype, num_layers, layer_stride, num_blocks,
                    block_size, num_kv_heads, head_dim, k_scales, v_scales, scale_layer_stride, src_pages,
                    dst_pages, index_type, 1, num_pairs, true, invalid_count, stream);
}

extern "C" int mkv_move_kv_rows(void* k_cache, void* v_cache, int32_t cache_dtype, int32_t num_layers,
                                int64_t layer_stride, int64_t num_blocks, int32_t block_size,
                                int32_t num_kv_heads, int32_t head_dim, float* k_scales, float* v_scales,
                                int64_t scale_layer_stride, const void* src_slots, const void* dst_slots,
                                int32_t index_type, int32_t num_groups, int32_t moves_per_group,
                                int32_t* invalid_count, void* stream) {
  clear_error();
  return copy_units("mkv_move_kv_rows", k_cache, v_cache, cache_dtype, num_layers, layer_stride, num_blocks,
                    block_size, num_kv_heads, head_dim, k_scales, v_scales, scale_layer_stride, src_slots,
                    dst_slots, index_type, num_groups, moves_per_group, false, invalid_count, stream);
}
