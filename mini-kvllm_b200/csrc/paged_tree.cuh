// Shared parts of the attention for trees of drafted tokens over the paged cache:
// parameters, the device-side work schedule, and which cached tokens a row sees.
#pragma once

#include "mkv_common.cuh"

namespace mkv {
namespace tree {

struct Params {
  const void* q;
  int64_t q_st, q_sh;  // elements
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  int64_t num_blocks;
  int block_size;
  const void* bt;
  int64_t bt_sb;
  int max_blocks, bt_i64;
  const void* ctx;
  const void* cu;
  int ctx_i64, cu_i64;
  const uint64_t* mask;  // (total_q, mask_words), row stride in words
  int64_t mask_st;
  int mask_words;
  int num_seqs, num_heads, num_kv_heads, head_dim, group;
  int64_t total_q;
  int unit_cost;  // of the schedule, in token tiles
  long long wait_limit;  // clocks that a wait may take
  float qk_scale_log2;
  const float* k_scale;   // per-tensor scales of e4m3 pages, or null
  const float* v_scale;
  const float* k_scales;  // per-(page, row, kv head) scales of 8-bit pages, or null
  const float* v_scales;
  void* out;
  int64_t o_st, o_sh;  // elements
  bool zero_rest;      // rows of no sequence become 0 (otherwise they are left)
  // split units: partial sums (2 slots per CTA) and one descriptor per CTA
  float* part_acc;  // [slot][row][head_dim], relative to the row's partial maximum
  float2* part_ml;  // [slot][row] = (maximum in the exp2 domain, sum)
  int4* desc;       // [cta][2]
};

__device__ __forceinline__ int64_t ld_idx(const void* p, int i64, int64_t i) {
  return i64 ? __ldg(reinterpret_cast<const int64_t*>(p) + i)
             : (int64_t)__ldg(reinterpret_cast<const int32_t*>(p) + i);
}

// A sequence of the batch: query rows [q0, q0 + nodes), cached tokens [0, len), the last
// `nodes` of them the tree's own (from `prefix` on).
struct Seq {
  int64_t q0;
  int nodes, len, prefix;
};
static __device__ __noinline__ Seq load_seq(const Params& p, int b) {
  Seq s;
  int64_t a = ld_idx(p.cu, p.cu_i64, b), e = ld_idx(p.cu, p.cu_i64, b + 1);
  a = min(max(a, (int64_t)0), p.total_q);
  e = min(max(e, (int64_t)0), p.total_q);
  s.q0 = a;
  s.nodes = e > a ? (int)(e - a) : 0;
  const int64_t ctx = ld_idx(p.ctx, p.ctx_i64, b);
  const int64_t cap = (int64_t)p.max_blocks * p.block_size;  // at most 2^31 - 1024 (checked on the host)
  s.len = (int)max(min(ctx, cap), (int64_t)0);
  s.prefix = (int)max(min(ctx - s.nodes, (int64_t)s.len), (int64_t)0);
  return s;
}

// Page of logical block blk of sequence b, or -1 (entry -1 or outside the cache).
__device__ __forceinline__ int64_t load_page(const Params& p, int b, int blk) {
  const int64_t page = ld_idx(p.bt, p.bt_i64, (int64_t)b * p.bt_sb + blk);
  return (page >= 0 && page < p.num_blocks) ? page : -1;
}

// The same in two steps: the entry as it lies in memory, loaded well before it is used (with
// nothing that waits for it), and the page that it means.
struct Entry {
  uint32_t lo, hi;
};
__device__ __forceinline__ Entry load_entry(const Params& p, int b, int blk) {
  const int64_t i = (int64_t)b * p.bt_sb + blk;
  Entry e;
  if (p.bt_i64) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p.bt) + i);
    e.lo = v.x;
    e.hi = v.y;
  } else {
    e.lo = __ldg(reinterpret_cast<const uint32_t*>(p.bt) + i);
    e.hi = 0;
  }
  return e;
}
__device__ __forceinline__ void prefetch_entry(const Params& p, int b, int blk) {
  const char* at = reinterpret_cast<const char*>(p.bt) + (((int64_t)b * p.bt_sb + blk) << (p.bt_i64 ? 3 : 2));
  asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
}
__device__ __forceinline__ int64_t page_of(const Params& p, Entry e) {
  const int64_t page = p.bt_i64 ? (int64_t)(((uint64_t)e.hi << 32) | e.lo) : (int64_t)(int32_t)e.lo;
  return (page >= 0 && page < p.num_blocks) ? page : -1;
}

// Visibility of the 32 tokens t0 .. t0 + 31 for one query row (bit i: token t0 + i): all of
// the prefix, the tree's nodes by the row's mask, nothing from len on.
// mask0: the row's first word, in hand.
__device__ __forceinline__ uint32_t visible32(const Seq& s, const uint64_t* mask_row, uint64_t mask0, int mask_words,
                                              int t0) {
  const int in = s.len - t0;  // tokens that exist
  if (in <= 0) return 0u;
  uint32_t v = in >= 32 ? 0xffffffffu : (1u << in) - 1u;
  const int j0 = t0 - s.prefix;  // node of bit 0
  if (j0 <= -32) return v;
  const int first = j0 < 0 ? 0 : j0;
  uint64_t bits = 0;
  if (first < 64) bits = mask0 >> first;
  else if ((first >> 6) < mask_words) bits = __ldg(mask_row + (first >> 6)) >> (first & 63);
  if ((first & 63) > 32 && (first >> 6) + 1 < mask_words)
    bits |= __ldg(mask_row + (first >> 6) + 1) << (64 - (first & 63));
  uint32_t t = (uint32_t)bits;
  if (j0 < 0) t = (t << -j0) | ((1u << -j0) - 1u);
  return v & t;
}

// ---------------------------------------------------------------- work schedule
// Work items are (sequence, kv head, tile of RT query rows, tile of KT tokens), in this
// order; a unit is a run of all token tiles of one row tile, followed by unit_cost items that
// stand for what a unit costs besides its tiles. CTA c of n takes items
// [c W / n, (c + 1) W / n): equal work whatever the lengths, known on the device alone. A unit
// that ends inside a CTA's share is written there whole; the parts of a unit that crosses
// shares go to partial slots (2 c + 1: the part that starts a unit, 2 c: any later one) and are
// joined by the combine kernel, which takes its orders from desc[c]: the first CTA that
// continues a unit gives the number of its parts, its kv head and first row, and the rows and
// the first query row of its sequence.
struct Unit {
  int b, kvh, mt;     // sequence, kv head, row tile
  int k0, k1, tiles;  // token tiles taken here, and of the whole unit
  Seq s;
};

// a / b of non-negative numbers, in 32 bits where both fit (64-bit division is a long call).
static __device__ __noinline__ int64_t quot(int64_t a, int64_t b) {
  if (((uint64_t)a | (uint64_t)b) >> 32 == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

template <int RT, int KT>
__device__ __forceinline__ int64_t items_of(const Params& p, const Seq& s, int& mt, int& kt) {
  mt = (int)(((int64_t)s.nodes * p.group + RT - 1) / RT);
  kt = max(1, (s.len + KT - 1) / KT);
  return (int64_t)p.num_kv_heads * mt * (kt + p.unit_cost);
}

struct Walk {
  int64_t left;    // items of this CTA not yet taken
  int b, kvh, mt, k;  // the next one
  int mts, kts;    // row and token tiles of sequence b
  Seq s;
};

// Finds CTA c's share. Block-collective over NT threads, with kBeginWords(NT) words of
// shared memory that are free again after the caller's next barrier; writes desc[c]. False
// when the CTA has nothing to do.
constexpr int kBeginWords(int nt) { return nt / 32 + 2; }
template <int RT, int KT, int NT>
__device__ bool begin(const Params& p, int c, int n, long long* red, Walk& w) {
  long long* found = red + NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // inclusive scan of one chunk of sequences; returns this thread's inclusive sum, `sum` the chunk's
  auto scan = [&](long long x, long long& sum) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += v;
    }
    __syncthreads();
    if (lane == 31) red[warp] = x;
    __syncthreads();
    sum = 0;
#pragma unroll 1
    for (int i = 0; i < NT / 32; ++i) {
      if (i < warp) x += red[i];
      sum += red[i];
    }
    return x;
  };
  auto items = [&](int b) -> long long {
    if (b >= p.num_seqs) return 0;
    int mt, kt;
    return items_of<RT, KT>(p, load_seq(p, b), mt, kt);
  };
  long long total = 0, mine = 0, incl = 0, sum;
#pragma unroll 1
  for (int base = 0; base < p.num_seqs; base += NT) {
    mine = items(base + tid);
    incl = scan(mine, sum);
    total += sum;
  }
  if (n > total) n = (int)total;  // every CTA that works has an item
  if (tid == 0) p.desc[2 * c] = make_int4(0, 0, 0, 0);
  if (c >= n) return false;
  const int64_t s0 = quot((int64_t)c * total, n), s1 = quot((int64_t)(c + 1) * total, n);
  long long before = 0;
#pragma unroll 1
  for (int base = 0; base < p.num_seqs; base += NT) {
    if (p.num_seqs > NT) {  // otherwise the first scan still holds
      mine = items(base + tid);
      incl = scan(mine, sum);
    }
    const long long i1 = before + incl;
    if (mine > 0 && i1 - mine <= s0 && s0 < i1) {
      found[0] = base + tid;
      found[1] = s0 - (i1 - mine);
    }
    before += sum;
    if (before > s0) break;
  }
  __syncthreads();
  w.left = s1 - s0;
  w.b = (int)found[0];
  const int64_t off = found[1];
  w.s = load_seq(p, w.b);
  items_of<RT, KT>(p, w.s, w.mts, w.kts);
  const int per = w.kts + p.unit_cost;
  const int64_t i = quot(off, per);
  w.k = (int)(off - i * per);
  w.kvh = (int)quot(i, w.mts);
  w.mt = (int)(i - (int64_t)w.kvh * w.mts);
  const int64_t unit0 = s0 - w.k;  // first item of the unit that s0 lies in
  if (w.k >= w.kts) {  // behind its tiles
    w.left -= per - w.k;
    w.k = w.kts;
  } else if (tid == 0 && w.k > 0 && quot((int64_t)(c - 1) * total, n) <= unit0) {
    // this CTA is the first to continue the unit: parts from CTA c - 1 to the one holding its last item
    const int64_t last = quot((unit0 + w.kts) * n + total - 1, total) - 1;
    p.desc[2 * c + 1] = make_int4((int)(w.s.q0 >> 32), (int)w.s.q0, 0, 0);
    p.desc[2 * c] = make_int4((int)(last - c + 2), w.kvh, w.mt * RT, w.s.nodes * p.group);
  }
  return true;
}

// The next unit, or the part of it that falls into this CTA's share.
template <int RT, int KT>
__device__ __forceinline__ bool next(const Params& p, Walk& w, Unit& u) {
  if (w.left <= 0) return false;
  if (w.k == w.kts) {  // on to the next unit
    w.k = 0;
    if (++w.mt == w.mts) {
      w.mt = 0;
      if (++w.kvh == p.num_kv_heads) {
        w.kvh = 0;
#pragma unroll 1
        do {  // sequences without nodes have no units
          w.s = load_seq(p, ++w.b);
          items_of<RT, KT>(p, w.s, w.mts, w.kts);
        } while (w.mts == 0);
      }
    }
  }
  u.b = w.b;
  u.s = w.s;
  u.kvh = w.kvh;
  u.mt = w.mt;
  u.k0 = w.k;
  u.tiles = w.kts;
  u.k1 = (int)min((int64_t)w.kts, w.k + w.left);
  w.left -= u.k1 - u.k0;
  if (u.k1 == w.kts) w.left -= p.unit_cost;
  w.k = u.k1;
  return true;
}

// Partial slot of a unit's part, -1 for a whole unit.
__device__ __forceinline__ int slot_of(const Unit& u, int c) {
  if (u.k0 == 0 && u.k1 == u.tiles) return -1;
  return 2 * c + (u.k0 == 0 ? 1 : 0);
}

// Sum that a part stores for a row whose visible scores were all -inf (0 / 0 where no other
// part has a finite one), as opposed to a row that saw nothing (0).
constexpr float kSeenInf = -1.0f;

// What a CTA gives when one of its waits has run out: NaN in every row of its share (in the partial
// sums of the units that it has a part of, which the join carries into the rows). Block-collective,
// called when nothing of the CTA is in flight any more; red as for begin().
template <int RT, int KT, int NT, typename QT>
__device__ __noinline__ void give_up(const Params& p, long long* red) {
  Walk w;
  if (!begin<RT, KT, NT>(p, blockIdx.x, gridDim.x, red, w)) return;
  Unit u;
  while (next<RT, KT>(p, w, u)) {
    const int rows = (int)min((int64_t)RT, (int64_t)u.s.nodes * p.group - (int64_t)u.mt * RT);
    const int slot = slot_of(u, blockIdx.x);
    for (int r = threadIdx.x >> 5; r < rows; r += NT / 32) {  // a warp per row
      const int lane = threadIdx.x & 31;
      if (slot >= 0) {
        if (lane == 0) p.part_ml[(int64_t)slot * RT + r] = make_float2(-INFINITY, NAN);
        continue;
      }
      const int R = u.mt * RT + r, node = R / p.group;
      QT* o = reinterpret_cast<QT*>(p.out) + (u.s.q0 + node) * p.o_st +
              (int64_t)(u.kvh * p.group + R - node * p.group) * p.o_sh;
      for (int d = lane; d < p.head_dim; d += 32) o[d] = from_f32<QT>(NAN);
    }
  }
}

// ---------------------------------------------------------------- host side
struct Workspace {
  size_t acc, ml, desc, total;  // offsets and size in bytes
};
Workspace workspace(int ctas, int rows, int head_dim);

// Clocks that a wait in the kernels may take (mkv_set_wait_limit).
int64_t wait_limit();

// tcgen05 variant (paged_tree_tc.cu): whether it takes the call, and its launch.
constexpr int kTcRows = 128;
bool tc_supported(const Params& p, int q_dtype, int cache_dtype);
int launch_tc(const Params& p, int q_dtype, int cache_dtype, int ctas, cudaStream_t stream);

}  // namespace tree
}  // namespace mkv
