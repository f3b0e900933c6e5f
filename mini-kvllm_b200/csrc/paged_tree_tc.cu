// Tree attention on the 5th-generation tensor cores: 16-bit queries, head_dim 64 or 128, pages of
// a power of two >= 8 tokens; caches in the query's dtype, e4m3 or int8.
//
// A persistent CTA per SM takes an even share of the token tiles (paged_tree.cuh). A unit is
// 128 query rows (node, GQA head) of one kv head; rows sit on TMEM lanes, so a row's maximum
// and sum need no exchange. Token tiles of 128 alternate between two streams, each with its
// own S / P buffer, its own accumulator O and its own warpgroup, running maximum and sum, so
// that one stream's softmax runs while the other's products do; the two are joined once per
// unit. TMEM: S0 | S1 | O0 | O1, 128 columns each, P (16 bits) over the first half of S.
//   warp 0      producer: K and V tiles by TMA (one box per page, 128-byte swizzle) into rings
//   warp 1      MMA issuer: S = Q K^T, O += P V (P from TMEM, V as it lies in its pages)
//   warps 2-3   stage the rows of Q, a unit ahead of the products (two buffers)
//   warps 4-11  softmax of stream 0 (4-7) and 1 (8-11); at a unit's end they join the streams
//               and write the output, while the products of the next unit start
//   warps 12-15 8-bit caches: converters of the raw tiles to f16 (exact) for the MMAs
// K/V bytes are read once per unit of 128 rows; with fewer rows the tensor core's work is
// padded, which costs nothing while the tile's bytes take longer to arrive (bf16: 64 KB a
// tile, 1.5 us of an SM's share of HBM; its two products 0.55 us).
//
// Measured (B200, device time of the call with its combine, short replays): bf16, 48 sequences of
// 1-8k tokens, 8-32 nodes, 32/8 heads 168-172 us, 5.4 TB/s (0.83 of the copy rate; 201 us where calls
// follow one another for seconds, under the power cap), DRAM reads 0.94 GB = K and V once; e4m3,
// 12 x 32k, 32 nodes 241-246 us, 840 TFLOP/s, tensor pipe 40 % and exponentials 40 % busy: a tile
// takes 2500 clocks; the MMA issuer is busy for 1375 of them, the converters for 2100 (890 convert,
// the rest are fences, arrivals and table lookups), the exponentials take 1050, in a chain that two
// streams overlap by half; int8 with row scales, 19 x 1-5k over 16-token pages 78 us: 2.0 us a tile
// (24 a CTA) and 28 us outside the tiles. Two streams, not one shared accumulator or half a tile per warpgroup: both
// measured slower (250-270 us against 319 and 391 for e4m3).
//
// What a row must not see: scores of hidden tokens are replaced by -inf before the maximum.
// Values meet P = 0 there, and 0 x inf is NaN, so rows of V that do not exist (past the
// context, missing pages) are zeroed in shared memory, and a tree's own rows, which some see
// and others do not, are searched for infinities and NaN: those are zeroed too, and added in
// at the end to the rows that see them.
//
// Every wait is bounded (mkv_set_wait_limit); a role that gives up raises the abort flag, the
// others stop, loads and MMAs in flight are waited for, TMEM is freed, and the CTA's rows become
// NaN (give_up), so that the failure is seen.
#include <cuda.h>

#include <type_traits>

#include "paged_tree.cuh"
#include "sm100.cuh"

namespace mkv {
namespace tree {
namespace {
using namespace sm100;

constexpr int kRows = kTcRows, kTile = 128;
constexpr int BLK = 128 * 128;  // 128 rows x 128 bytes: 64 columns of a 16-bit tile
constexpr uint32_t kTmemCols = 512, kOCol = 256;
constexpr int kSickSlots = 4;
constexpr int kWide = 6;     // binades of V scales in a tile beyond which a row takes an exponent of its own
constexpr float kHold = 60;  // binades that O may lie above its unit

// kByte: 8-bit cache; kTok: with per-(token, head) scales.
template <bool kByte, bool kTok, int kD>
struct Layout {
  static constexpr int TILE = kD / 64 * BLK;  // a 16-bit tile
  static constexpr int RAW = kTile * kD;      // an 8-bit one
  static constexpr int kThreads = kByte ? 512 : 384;
  // 16-bit K and V tiles. 8-bit: one K tile is enough, as the next one is converted while the
  // tensor core works on the values of the tile before
  static constexpr int kKS = kByte ? 1 : 3;
  static constexpr int kVS = 2;
  static constexpr int kRS = kByte ? 2 : 0;  // raw 8-bit tiles (K and V)
  static constexpr int Q0 = 0;               // [2]; a free one carries the streams' joint statistics
  static constexpr int K0 = Q0 + 2 * TILE;
  static constexpr int V0 = K0 + kKS * TILE;
  static constexpr int R0 = V0 + kVS * TILE;
  static constexpr int SC0 = R0 + kRS * 2 * RAW;             // [V stage][K scale, V factor][128]
  static constexpr int QE0 = SC0 + (kTok ? kVS * 2 * kTile * 4 : 0);  // [2][128] exponents of Q's rows
  static constexpr int ONE0 = QE0 + (kByte ? 2 * kRows : 0);          // [128] ones: K scales of a masked tile
  static constexpr int BAR0 = ONE0 + (kTok ? kTile * 4 : 0);
  static constexpr int NBAR = 2 * kKS + 2 * kVS + 2 * kRS + 4 + 2 + 2 + 1 + 2 + 1 + 1;
  static constexpr int MISC0 = BAR0 + NBAR * 8;              // tmem base, abort, sick[4], exponents[2], ranges[2][4]
  static constexpr int BYTES = MISC0 + 64;
  static_assert(BYTES <= 232448, "shared memory per CTA");
  static_assert(kBeginWords(kThreads) * 8 <= TILE, "the schedule's scratch lies in the first K stage");
};

// A wait that has not been met at once; out of line, as the roles' code should stay small
// (instructions that one role fetches push out another's).
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, const volatile int* abort, long long limit) {
  return mbar_wait(bar, parity, abort, limit);
}

// 16 bytes of an 8-bit row -> 16 f16 values, exact.
template <typename CT>
__device__ __forceinline__ void to_f16x16(const uint4 raw, uint32_t (&h)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (std::is_same<CT, int8_t>::value) {
      h[2 * j] = s8x2_to_f16x2((uint16_t)w[j]);
      h[2 * j + 1] = s8x2_to_f16x2((uint16_t)(w[j] >> 16));
    } else {
      e4m3x4_to_f16x2x2(w[j], h[2 * j], h[2 * j + 1]);
    }
  }
}

// Clears the infinities and NaN of a row of 16-bit values in a tile (kExp: the type's exponent
// bits; `bytes` of them from `row`, the other 64 columns BLK further on); true when there were
// any. Out of line, like wait_on: few tiles hold nodes.
template <uint32_t kExp>
__device__ __noinline__ bool clear_sick(uint8_t* row, int bytes) {
  bool sick = false;
#pragma unroll 1
  for (int c = 0; c < bytes; c += 16) {
    uint4* at = reinterpret_cast<uint4*>(row + (c >> 7) * BLK + (c & 127));
    uint32_t w[4] = {at->x, at->y, at->z, at->w};
    bool here = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t keep = ((w[e] & kExp) == kExp ? 0u : 0x0000ffffu) |
                            ((w[e] >> 16 & kExp) == kExp ? 0u : 0xffff0000u);
      here |= keep != 0xffffffffu;
      w[e] &= keep;
    }
    if (here) *at = make_uint4(w[0], w[1], w[2], w[3]);
    sick |= here;
  }
  return sick;
}

__device__ __forceinline__ float pow2f(int e) {  // 2^e, -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

template <typename QT, typename CT, bool kTok, int kD>
__global__ void __launch_bounds__((Layout<sizeof(CT) == 1, kTok, kD>::kThreads), 1)
paged_tree_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap) {
  constexpr bool kByte = sizeof(CT) == 1;
  using L = Layout<kByte, kTok, kD>;
  constexpr int TILE = L::TILE;
  using MT = typename std::conditional<kByte, f16, QT>::type;  // operands of the MMAs
  // f16 weights: 2^6 above the reference, so that they stay normal down to 2^-20 of the
  // largest (below 2^-31 of it they are 0: up to that times the value is lost of a token, which
  // counts where the heavy tokens' values are 0); with the lazy reference (2^8) and a scale factor
  // below 2 they end below 2^15.
  constexpr float kBias = std::is_same<MT, f16>::value ? 6.0f : 0.0f;
  constexpr bool kToF16 = kByte && std::is_same<QT, bf16>::value;  // Q changes its type
  constexpr int kKS = L::kKS, kVS = L::kVS, kRS = kByte ? L::kRS : 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::BAR0);
  uint64_t* kempty = kfull + kKS;
  uint64_t* vfull = kempty + kKS;
  uint64_t* vempty = vfull + kVS;
  uint64_t* rfull = vempty + kVS;
  uint64_t* rempty = rfull + L::kRS;
  uint64_t* qfull = rempty + L::kRS;
  uint64_t* qempty = qfull + 2;
  uint64_t* sfull = qempty + 2;
  uint64_t* pfull = sfull + 2;
  uint64_t* ofull = pfull + 2;
  uint64_t* xbar = ofull + 1;
  uint64_t* drain = xbar + 2;
  uint64_t* cbar = drain + 1;
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(smem + L::MISC0);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC0 + 4);
  volatile int* sick_s = reinterpret_cast<volatile int*>(smem + L::MISC0 + 8);
  volatile int* vexp_s = reinterpret_cast<volatile int*>(smem + L::MISC0 + 8 + 4 * kSickSlots);
  volatile uint32_t* vmax_s = reinterpret_cast<volatile uint32_t*>(smem + L::MISC0 + 16 + 4 * kSickSlots);
  int8_t* qexp_s = reinterpret_cast<int8_t*>(smem + L::QE0);
  float* scales_s = reinterpret_cast<float*>(smem + L::SC0);
  float* ones_s = reinterpret_cast<float*>(smem + L::ONE0);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kKS; ++s) {
      mbar_init(&kfull[s], kByte ? 4 : 1);
      mbar_init(&kempty[s], 1);
    }
    for (int s = 0; s < kVS; ++s) {
      mbar_init(&vfull[s], kByte ? 4 : 1);
      mbar_init(&vempty[s], 1);
    }
    for (int s = 0; s < L::kRS; ++s) {
      mbar_init(&rfull[s], 1);
      mbar_init(&rempty[s], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&qfull[b], 2);
      mbar_init(&qempty[b], 8);
      mbar_init(&sfull[b], 1);
      mbar_init(&pfull[b], 4);
      mbar_init(&xbar[b], 8);
    }
    mbar_init(ofull, 1);
    mbar_init(drain, 1);
    mbar_init(cbar, 4);
    *abort_flag = 0;
    for (int i = 0; i < kSickSlots; ++i) sick_s[i] = 0;
    fence_barrier_init();
  }
  if (kTok && tid < kTile) ones_s[tid] = 1.0f;
  if (warp == 1) tmem_alloc(tmem_base_s, kTmemCols);
  Walk walk;
  const bool work =
      begin<kRows, kTile, L::kThreads>(p, blockIdx.x, gridDim.x, reinterpret_cast<long long*>(smem + L::K0), walk);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_trigger();  // the combine kernel may be set up (it waits for this one's end)
  const uint32_t tmem = *tmem_base_s;
  if (!work) {
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  // a tile is loaded in segments of one page (or of kTile tokens of a larger page)
  const int seg_rows = p.block_size < kTile ? p.block_size : kTile;
  const int nseg = kTile / seg_rows;
  auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {  // warp-uniform
    bool done = mbar_try_wait(bar, phase & 1);
    if (!done) done = wait_on(bar, phase & 1, abort_flag, p.wait_limit);
    return __all_sync(0xffffffffu, done);
  };
  const int bs_log2 = 31 - __clz(p.block_size);
  // table entry of segment `lane` of tile t, and its page: -1 where it is missing or past the context
  auto seg_in = [&](const Unit& u, int t) -> bool { return lane < nseg && t * kTile + lane * seg_rows < u.s.len; };
  auto seg_entry = [&](const Unit& u, int t) -> Entry {
    Entry e{0xffffffffu, 0xffffffffu};
    if (seg_in(u, t)) e = load_entry(p, u.b, (t * kTile + lane * seg_rows) >> bs_log2);
    return e;
  };
  auto seg_page = [&](const Unit& u, int t, Entry e) -> int64_t { return seg_in(u, t) ? page_of(p, e) : -1; };
  Unit u = {};
  uint32_t g = 0;     // tiles of this CTA before the unit's
  uint32_t unit = 0;  // units before this one
  bool ok = p.wait_limit > 0;  // (0: no wait is allowed at all)

  if (warp == 0) {
    // ================================================================ producer
    if (lane == 0) {
      tma_prefetch_map(&kmap);
      tma_prefetch_map(&vmap);
    }
    uint32_t nk = 0, nv = 0;  // K and V tiles issued (8-bit: nk counts both)
    // loads the rows of tile t that exist, each lane its own segment (with pages of 16 tokens a tile is
    // 16 to 32 loads); the rest of the stage keeps what it held
    auto load = [&](const CUtensorMap* map, int t, int64_t page, uint32_t dst, uint64_t* bar) {
      if (page >= 0) {
        const int y = (int)(page * p.block_size) + ((t * kTile + lane * seg_rows) & (p.block_size - 1));
        tma_load_2d(dst + lane * seg_rows * (kByte ? kD : 128), map, u.kvh * kD, y, bar);
        if constexpr (!kByte && kD == 128) tma_load_2d(dst + BLK + lane * seg_rows * 128, map, u.kvh * kD + 64, y, bar);
      }
      __syncwarp();
    };
    auto seg_bytes = [&](int64_t page) -> uint32_t {  // of one tile
      return (uint32_t)__popc(__ballot_sync(0xffffffffu, page >= 0)) * (uint32_t)(seg_rows * kD * (int)sizeof(CT));
    };
#pragma unroll 1
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      int64_t page_v = -1;
      Entry next_e = seg_entry(u, u.k0);  // looked up one tile ahead
#pragma unroll 1
      for (int i = 0; i <= tiles && ok; ++i) {
        const int64_t page_k = i < tiles ? seg_page(u, u.k0 + i, next_e) : -1;
        if (i + 1 < tiles) next_e = seg_entry(u, u.k0 + i + 1);
        if (i + 8 < tiles && seg_in(u, u.k0 + i + 8))
          prefetch_entry(p, u.b, ((u.k0 + i + 8) * kTile + lane * seg_rows) >> bs_log2);
        if constexpr (kByte) {
          if (i == tiles) break;
          const uint32_t st = nk % kRS;
          if (!(ok = wait(&rempty[st], nk / kRS + 1))) break;
          const uint32_t bytes = 2 * seg_bytes(page_k);
          if (lane == 0) mbar_arrive_expect_tx(&rfull[st], bytes);
          __syncwarp();
          const uint32_t dst = smem_u32(smem + L::R0 + st * 2 * L::RAW);
          load(&kmap, u.k0 + i, page_k, dst, &rfull[st]);
          load(&vmap, u.k0 + i, page_k, dst + L::RAW, &rfull[st]);
          ++nk;
        } else {  // K one tile ahead of V, the order in which the products take them
          if (i < tiles) {
            const uint32_t st = nk % kKS;
            if (!(ok = wait(&kempty[st], nk / kKS + 1))) break;
            const uint32_t bytes = seg_bytes(page_k);
            if (lane == 0) mbar_arrive_expect_tx(&kfull[st], bytes);
            __syncwarp();
            load(&kmap, u.k0 + i, page_k, smem_u32(smem + L::K0 + st * TILE), &kfull[st]);
            ++nk;
          }
          if (i > 0) {
            const uint32_t st = nv % kVS;
            if (!(ok = wait(&vempty[st], nv / kVS + 1))) break;
            const uint32_t bytes = seg_bytes(page_v);
            if (lane == 0) mbar_arrive_expect_tx(&vfull[st], bytes);
            __syncwarp();
            load(&vmap, u.k0 + i - 1, page_v, smem_u32(smem + L::V0 + st * TILE), &vfull[st]);
            ++nv;
          }
          page_v = page_k;
        }
      }
    }
    if (!ok) *abort_flag = 1;
    __syncwarp();
    // loads in flight land before the CTA goes on to its end, whichever role gives up, and when (in a call
    // that runs well the last tile's products wait for the same loads)
    if (lane == 0) {
      if constexpr (kByte) {
        for (uint32_t k = nk > kRS ? nk - kRS : 0; k < nk; ++k) mbar_wait(&rfull[k % kRS], (k / kRS) & 1, nullptr);
      } else {
        for (uint32_t k = nk > kKS ? nk - kKS : 0; k < nk; ++k) mbar_wait(&kfull[k % kKS], (k / kKS) & 1, nullptr);
        for (uint32_t k = nv > kVS ? nv - kVS : 0; k < nv; ++k) mbar_wait(&vfull[k % kVS], (k / kVS) & 1, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ================================================================ MMA issuer
    constexpr uint32_t fmt = std::is_same<MT, bf16>::value ? 1u : 0u;
    constexpr uint32_t kIdQK = instr_desc(fmt, fmt, 0, 0, kRows, kTile);
    constexpr uint32_t kIdPV = instr_desc(fmt, fmt, 0, 1, kRows, kD);
    uint32_t ns[2] = {0, 0};  // tiles that each stream has had P for
    auto qk = [&](int i) -> bool {  // S[i & 1] = Q K(i)^T
      const uint32_t k = g + i, st = k % kKS;
      if (!wait(&kfull[st], k / kKS)) return false;
      tc_fence_after_sync();
      if (elect_one()) {
        const uint64_t qd = smem_desc(smem_u32(smem + L::Q0 + (unit & 1) * TILE), 16, 1024, kLayoutSw128);
        const uint64_t kd = smem_desc(smem_u32(smem + L::K0 + st * TILE), 16, 1024, kLayoutSw128);
#pragma unroll
        for (int c = 0; c < kD / 16; ++c) {  // 16 head_dim columns per MMA (descriptors count 16 bytes)
          const uint32_t off = ((c >> 2) * BLK + (c & 3) * 32) >> 4;
          mma_f16(tmem + (i & 1) * kTile, qd + off, kd + off, kIdQK, c > 0 ? 1u : 0u);
        }
        mma_commit(&sfull[i & 1]);
        mma_commit(&kempty[st]);
      }
      __syncwarp();
      return true;
    };
    auto pv = [&](int i) -> bool {  // O[i & 1] += P(i) V(i)
      const uint32_t v = g + i, st = v % kVS;
      if (!wait(&pfull[i & 1], ns[i & 1]) || !wait(&vfull[st], v / kVS)) return false;
      ++ns[i & 1];
      tc_fence_after_sync();
      if (elect_one()) {
        const uint64_t vd = smem_desc(smem_u32(smem + L::V0 + st * TILE), BLK, 1024, kLayoutSw128);
#pragma unroll
        for (int c = 0; c < kTile / 16; ++c)  // 16 tokens per MMA: 8 columns of P
          mma_f16_ts(tmem + kOCol + (i & 1) * kD, tmem + (i & 1) * kTile + 8 * c, vd + c * (2048 >> 4), kIdPV,
                     (i > 1 || c > 0) ? 1u : 0u);
        mma_commit(&vempty[st]);
      }
      __syncwarp();
      return true;
    };
#pragma unroll 1
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      ok = wait(&qfull[unit & 1], unit >> 1);
      // QK(0), QK(1), PV(0), QK(2), PV(1), ...: QK(i) is issued after PV(i - 2), which reads the P
      // that it overwrites; MMAs run in the order of issue, so its S being full also says that
      // PV(i - 2) is done
#pragma unroll 1
      for (int i = 0; i < tiles + 2 && ok; ++i) ok = (i < 2 || pv(i - 2)) && (i >= tiles || qk(i));
      if (ok && elect_one()) mma_commit(ofull);
      __syncwarp();
      g += tiles;
      ++unit;
    }
    if (!ok) *abort_flag = 1;
    if (elect_one()) {  // every MMA done before TMEM is freed
      mma_commit(drain);
      mbar_wait(drain, 0, nullptr);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ================================================================ rows of Q
    // (128-byte swizzle, two halves of 64 columns). A negative score scale
    // turns them around, so that the softmax has a positive one.
    bool flip = p.qk_scale_log2 < 0.0f;
    if (kByte && !kTok) flip = flip != (__ldg(p.k_scale) < 0.0f);
    const uint32_t sign = flip ? 0x80008000u : 0u;
#pragma unroll 1
    while (ok && next<kRows, kTile>(p, walk, u)) {
      if (!(ok = wait(&qempty[unit & 1], (unit >> 1) + 1))) break;
      const int rows = u.s.nodes * p.group - u.mt * kRows;
      // 16 bytes a lane; every load is in flight at once (behind the tiles' bytes a
      // load takes microseconds)
      constexpr int kLanes = kD / 8, kStep = 64 / kLanes;  // lanes of a row, rows of a round
      const int c = lane % kLanes, r0 = (32 / kLanes) * (warp - 2) + lane / kLanes;
      uint8_t* dst = smem + L::Q0 + (unit & 1) * TILE + (c >> 3) * BLK;
#pragma unroll 4
      for (int r = r0; r < kRows; r += kStep) {
        const int R = u.mt * kRows + min(r, rows - 1), node = R / p.group;
        const QT* src = reinterpret_cast<const QT*>(p.q) + (u.s.q0 + node) * p.q_st +
                        (int64_t)(u.kvh * p.group + R - node * p.group) * p.q_sh + c * 8;
        cp_async_16(smem_u32(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4)), src, r < rows ? 16 : 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      if (kToF16 || sign != 0) {
#pragma unroll 4
        for (int r = r0; r < kRows; r += kStep) {
          uint4* at = reinterpret_cast<uint4*>(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4));
          uint4 v = *at;
          float up = 1.0f;
          if constexpr (kToF16) {
            // bf16 rows become f16 times a power of two that puts the largest value at 2^14: exact
            // down to 2^-28 of it
            auto top = [](uint32_t w) {
              return fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u)));
            };
            float mx = fmaxf(fmaxf(top(v.x), top(v.y)), fmaxf(top(v.z), top(v.w)));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            int e = 0;
            if (mx > 0.0f) e = min(max(14 - ((int)(__float_as_uint(mx) >> 23) - 127), -100), 100);
            up = pow2f(e);
            if (c == 0) qexp_s[(unit & 1) * kRows + r] = (int8_t)e;
          }
          auto put = [&](uint32_t w) -> uint32_t {
            if constexpr (kToF16) w = pack2<f16>(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
            return w ^ sign;
          };
          *at = make_uint4(put(v.x), put(v.y), put(v.z), put(v.w));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&qfull[unit & 1]);
      ++unit;
    }
    if (!ok) *abort_flag = 1;
  } else if (warp < 12) {
    // ================================================================ softmax
    const int stream = (warp - 4) >> 2;       // also the half of the columns that it writes
    const int rt = 32 * (warp & 3) + lane;    // row = TMEM lane
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t sa = tmem + lane_base + stream * kTile, oa = tmem + lane_base + kOCol;
    uint32_t ns = 0;  // tiles that this stream has had
    float sc0 = p.qk_scale_log2;
    float vs0 = 1.0f;
    if (kByte && !kTok) {
      sc0 *= __ldg(p.k_scale);
      vs0 = __ldg(p.v_scale);
    }
    sc0 = fabsf(sc0);  // the rows of Q take a negative sign
#pragma unroll 1
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      const int R = u.mt * kRows + rt, rows_left = u.s.nodes * p.group - u.mt * kRows;
      const bool live = rt < rows_left;
      const bool warp_live = 32 * (warp & 3) < rows_left;
      const int node = live ? R / p.group : 0;
      const int64_t qrow = u.s.q0 + node;
      const int head = u.kvh * p.group + (live ? R - node * p.group : 0);
      const uint64_t* mask_row = p.mask + qrow * p.mask_st;
      const uint64_t mask0 = __ldg(mask_row);
      float sc = sc0;
      if constexpr (kToF16) {  // the row's power of two
        if (!(ok = wait(&qfull[unit & 1], unit >> 1))) break;
        sc *= pow2f(-(int)qexp_s[(unit & 1) * kRows + rt]);
      }
      if (sc < 1e-37f) sc = 1e-37f;  // not 0, so that a masked -inf stays one
      float m = -INFINITY, l = 0.0f;  // reference (exp2 domain) and sum of this stream
      // kTok: O holds values times 2^-vexp, its terms so far are below 2^hold times their number
      float vexp = 0.0f, hold = -INFINITY;
      bool seen = false;
      Entry next_e = seg_entry(u, u.k0 + stream);
#pragma unroll 1
      for (int i = stream; i < tiles && ok; i += 2) {
        const int t0 = (u.k0 + i) * kTile;
        const uint32_t st = (g + i) % kVS, vph = (g + i) / kVS;
        const int64_t page = seg_page(u, u.k0 + i, next_e);
        if (i + 2 < tiles) next_e = seg_entry(u, u.k0 + i + 2);
        // ---- what the row sees: everything but in tiles with tree nodes, an end or a missing page
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t want = __ballot_sync(0xffffffffu, lane < nseg && t0 + lane * seg_rows < u.s.len);
        const bool special = t0 + kTile > u.s.prefix || have != want;
        auto visible = [&](int h) -> uint32_t {  // tokens 32 h .. of the tile that the row sees
          uint32_t vis = visible32(u.s, mask_row, mask0, p.mask_words, t0 + 32 * h);
          if (have != want) {
            if (seg_rows >= 32) {
              if (!((have >> ((32 * h) / seg_rows)) & 1u)) vis = 0;
            } else {
#pragma unroll 1
              for (int b = 0; b < 32; b += seg_rows)
                if (!((have >> ((32 * h + b) / seg_rows)) & 1u)) vis &= ~(((1u << seg_rows) - 1u) << b);
            }
          }
          return vis;
        };
        if (!special) seen = true;
        if (!(ok = wait(&sfull[stream], ns))) break;  // also: PV of the stream's previous tile is done
        tc_fence_after_sync();
        const float* ksp = scales_s + st * 2 * kTile;
        float alpha = 1.0f;
        bool rescale = false;
        if (kByte && (kTok || special)) {  // the converters have written the tile's scales and flags
          if (!(ok = wait(&vfull[st], vph))) break;
        }
        float tile_exp = 0.0f, er = 0.0f;  // unit of the tile's V factors, and of this row's products
        bool wide = false;
        if constexpr (kTok) {
          const int e = vexp_s[st];
          tile_exp = er = (float)(e >> 1);
          wide = e & 1;
        }
        if (warp_live) {
          // 32 scores, times the tokens' K scales
          const float* kscale = ksp;
          auto scores = [&](int h, float (&v)[32]) {
            tmem_ld32(sa + 32 * h, v);
            if constexpr (kTok) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(kscale + 32 * h + e);
                v[e] *= k4.x;
                v[e + 1] *= k4.y;
                v[e + 2] *= k4.z;
                v[e + 3] *= k4.w;
              }
            }
          };
          if (special) {  // the mask is put into S (and the K scales with it), so that the loops below have none
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
              float v[32];
              scores(h, v);
              const uint32_t vis = visible(h);
              seen |= vis != 0u;
              uint32_t w[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) w[e] = (vis >> e) & 1u ? __float_as_uint(v[e]) : 0xff800000u;
              tmem_st32(sa + 32 * h, w);
            }
            tmem_wait_st();
            if constexpr (kTok) kscale = ones_s;
          }
          // the tile's maximum, then P, 32 columns at a time (S is read twice: that costs less
          // than the registers to hold it, whose spills miss an L1 that shared memory has
          // taken; and short loops keep the roles' code in the instruction cache)
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {
            float v[32];
            scores(h, v);
#pragma unroll
            for (int e = 0; e < 32; e += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) mx[k] = fmax3(mx[k], v[e + k], v[e + 4 + k]);
          }
          // the reference moves only when a row's maximum has grown by more than 2^8, or is its first
          const float mt = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]) * sc;
          const bool need = mt > m + 8.0f;
          const float m_new = need ? mt : m;
          const float a2 = need ? exp2f(m - m_new) : 1.0f;  // 0 when m was -inf
          if constexpr (kTok) {
            // The tile's V factors are below 2, but where some are far below (wide) those that the row
            // does not see, or that hardly weigh, must not push its products into the subnormals of f16:
            // its own unit puts the largest product near 2^kBias. O may end up to 2^kHold above that.
            if (wide) {
              float top = -INFINITY;  // log2 of the largest weight times factor, rounded up
#pragma unroll 1
              for (int h = 0; h < 4; ++h) {
                float v[32];
                scores(h, v);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const int fx = (int)(__float_as_uint(ksp[kTile + 32 * h + e]) >> 23 & 255u) - 126;
                  top = fmaxf(top, fmaf(v[e], sc, (float)fx));
                }
              }
              er = top == -INFINITY ? vexp : er + fminf(fmaxf(floorf(top - m_new), -120.0f), 120.0f);
            }
            if (need) hold -= m_new - m;
            er = fmaxf(er, hold - kHold);
            hold = fmaxf(hold, er);
            alpha = exp2f(vexp - er + (need ? m - m_new : 0.0f));
            rescale = vexp != er;
            vexp = er;
          }
          const float nref = kBias - (m_new == -INFINITY ? 0.0f : m_new);
          const uint64_t sc2 = f2_pack(sc, sc), nref2 = f2_pack(nref, nref);
          uint64_t acc[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
          // (own: the row's unit is not the tile's)
          auto weights = [&](auto own, float factor) {
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
              float v[32];
              uint32_t w[16];
              scores(h, v);
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float x0, x1;
                f2_unpack(f2_fma(f2_pack(v[2 * e], v[2 * e + 1]), sc2, nref2), x0, x1);
                float p0 = ex2_approx(x0), p1 = ex2_approx(x1);  // 0 where masked
                acc[e & 1] = f2_add(acc[e & 1], f2_pack(p0, p1));
                if constexpr (kTok) {
                  float2 f = *reinterpret_cast<const float2*>(ksp + kTile + 32 * h + 2 * e);
                  if constexpr (decltype(own)::value) {
                    f.x *= factor;
                    f.y *= factor;
                  }
                  p0 *= f.x;
                  p1 *= f.y;
                }
                w[e] = pack2<MT>(p0, p1);
              }
              tmem_st16u(sa + 16 * h, w);  // over columns of S that have been read
            }
          };
          if (kTok && __any_sync(0xffffffffu, er != tile_exp))
            weights(std::true_type{}, exp2f(fminf(fmaxf(tile_exp - er, -126.0f), 120.0f)));
          else
            weights(std::false_type{}, 1.0f);
          float s0, s1, s2, s3;
          f2_unpack(acc[0], s0, s1);
          f2_unpack(acc[1], s2, s3);
          const float sum = (s0 + s1) + (s2 + s3);
          if (i > stream) {  // O holds something
            rescale = __any_sync(0xffffffffu, rescale || need);
            if constexpr (!kTok) alpha = a2;
          } else {
            rescale = false;
          }
          m = m_new;
          l = fmaf(l, a2, sum);
          if (rescale) {
#pragma unroll 1
            for (int c = 0; c < kD / 16; ++c) {
              float v[16];
              tmem_ld16(oa + stream * kD + 16 * c, v);
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] *= alpha;
              tmem_st16(oa + stream * kD + 16 * c, v);
            }
          }
          tmem_wait_st();
        }
        if (!kByte && special) {
          // rows of V that do not exist: zeros; a tree node's: without infinities and NaN
          if (!(ok = wait(&vfull[st], vph))) break;
          const int t = t0 + rt;
          const bool exists = t < u.s.len && ((have >> (rt / seg_rows)) & 1u);
          uint8_t* vrow = smem + L::V0 + st * TILE + rt * 128;
          if (!exists) {
#pragma unroll 4
            for (int k = 0; k < kD / 8; ++k)
              *reinterpret_cast<uint4*>(vrow + (k >> 3) * BLK + (k & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          } else if (t >= u.s.prefix) {
            const bool sick = clear_sick<std::is_same<QT, bf16>::value ? 0x7f80u : 0x7c00u>(vrow, kD * 2);
            if (sick) sick_s[unit % kSickSlots] = (int)unit + 1;
          }
          fence_proxy_async_smem();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[stream]);
        ++ns;
      }
      // ---- the unit's end: the streams exchange their references and sums
      if (ok) ok = wait(ofull, unit);
      if (!ok) break;
      tc_fence_after_sync();
      // the products of this unit are done with its Q: its buffer takes the statistics
      float4* stats = reinterpret_cast<float4*>(smem + L::Q0 + (unit & 1) * TILE);
      stats[stream * kRows + rt] = make_float4(m, l, vexp, seen ? 1.0f : 0.0f);
      __syncwarp();
      if (lane == 0) mbar_arrive(&xbar[0]);
      if (!(ok = wait(&xbar[0], unit))) break;
      const float4 xs = stats[(stream ^ 1) * kRows + rt];
      __syncwarp();
      if (lane == 0) mbar_arrive(&qempty[unit & 1]);
      if (warp_live) {
        const float x[4] = {xs.x, xs.y, xs.z, xs.w};
        const bool both = tiles > 1;
        const float M = both ? fmaxf(m, x[0]) : (stream == 0 ? m : x[0]);
        const float base = M == -INFINITY ? 0.0f : M;
        const float am = exp2f(m - base), ax = exp2f(x[0] - base);
        // (a stream without a tile has m = -inf and l = 0)
        const float lm = stream == 0 || both ? am * l : 0.0f, lx = stream == 1 || both ? ax * x[1] : 0.0f;
        float Ls = lm + lx;
        const bool any = seen || x[3] != 0.0f;
        const float a0 = vs0 * (stream == 0 ? am * exp2f(vexp) : ax * exp2f(x[2]));
        const float a1 = vs0 * (stream == 1 ? am * exp2f(vexp) : ax * exp2f(x[2]));
        const int slot = slot_of(u, blockIdx.x);
        float inv = 1.0f;
        if (slot < 0) inv = Ls == 0.0f ? (any ? NAN : 0.0f) : 1.0f / Ls;
        QT* dst = reinterpret_cast<QT*>(p.out) + qrow * p.o_st + (int64_t)head * p.o_sh + stream * (kD / 2);
        float* part = p.part_acc + ((int64_t)(slot < 0 ? 0 : slot) * kRows + rt) * kD + stream * (kD / 2);
        const bool sick = sick_s[unit % kSickSlots] == (int)unit + 1;
#pragma unroll 1
        for (int c = 0; c < kD / 64; ++c) {
          float v[32];
          tmem_ld32(oa + stream * (kD / 2) + 32 * c, v);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] *= a0;
          if (both) {
            float y[32];
            tmem_ld32(oa + kD + stream * (kD / 2) + 32 * c, y);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = fmaf(y[e], a1, v[e]);
          }
          if (!live) continue;
          if (slot < 0) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(dst + 32 * c + e) =
                  make_uint4(pack2<QT>(v[e] * inv, v[e + 1] * inv), pack2<QT>(v[e + 2] * inv, v[e + 3] * inv),
                             pack2<QT>(v[e + 4] * inv, v[e + 5] * inv), pack2<QT>(v[e + 6] * inv, v[e + 7] * inv));
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + 32 * c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
        if (sick && live) {  // infinities and NaN of the nodes that the row sees, added to what was stored
#pragma unroll 1
          for (int t = max(u.s.prefix, u.k0 * kTile); t < min(u.s.len, u.k1 * kTile); ++t) {
            const int64_t page = load_page(p, u.b, t >> bs_log2);
            if (page < 0 || !(visible32(u.s, mask_row, mask0, p.mask_words, t) & 1u)) continue;
            const int64_t row = (page * p.block_size + (t & (p.block_size - 1))) * p.num_kv_heads + u.kvh;
            const CT* vr = reinterpret_cast<const CT*>(p.v_cache) + row * kD + stream * (kD / 2);
            const float f = kTok ? __ldg(p.v_scales + row) : 1.0f;
#pragma unroll 1
            for (int e = 0; e < kD / 2; ++e) {
              const float x2 = to_f32(vr[e]) * f;
              if (isfinite(x2)) continue;
              if (slot < 0) dst[e] = from_f32<QT>(to_f32(dst[e]) + x2);
              else part[e] += x2;
            }
          }
        }
        if (slot >= 0 && stream == 0 && live)
          p.part_ml[(int64_t)slot * kRows + rt] = make_float2(M, Ls == 0.0f && any ? kSeenInf : Ls);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&xbar[1]);  // O has been read
      if (!(ok = wait(&xbar[1], unit))) break;
      tc_fence_after_sync();
      g += tiles;
      ++unit;
    }
    if (!ok) *abort_flag = 1;
  } else if (kByte && warp >= 12) {
    // ================================================================ converters
    // Thread r converts row r (token t0 + r) of K and V. Rows that do not exist become zeros.
    const int r = 32 * (warp - 12) + lane;
    int vexp = 0;
    // table entry of token t, and its (page, row, head) index in the cache (-1: none)
    auto tok_entry = [&](int t) -> Entry {
      Entry e{0xffffffffu, 0xffffffffu};
      if (t < u.s.len) e = load_entry(p, u.b, t >> bs_log2);
      return e;
    };
    auto row_of = [&](int t, Entry e) -> int64_t {
      const int64_t page = t < u.s.len ? page_of(p, e) : -1;
      if constexpr (!kTok) return page;  // (whether there is one is all that matters)
      return page < 0 ? -1 : (page * p.block_size + (t & (p.block_size - 1))) * p.num_kv_heads + u.kvh;
    };
    auto convert = [&](const uint8_t* src, uint8_t* dst, bool valid) {
      uint8_t* drow = dst + r * 128;
      uint4 raw[kD / 16];  // all loads first: a store in between would hold the next one back
      const int turn = kD == 128 ? r & 7 : (r >> 1) & 3;  // the swizzle of 128- and of 64-byte rows
#pragma unroll
      for (int c = 0; c < kD / 16; ++c) raw[c] = *reinterpret_cast<const uint4*>(src + r * kD + ((c ^ turn) << 4));
#pragma unroll
      for (int c = 0; c < kD / 16; ++c) {
        uint32_t h[8];
        if (!valid) raw[c] = make_uint4(0u, 0u, 0u, 0u);
        to_f16x16<CT>(raw[c], h);
        const int cc = (c & 3) * 2;  // columns 16c ..: half c / 4, chunks cc and cc + 1
        *reinterpret_cast<uint4*>(drow + (c >> 2) * BLK + ((cc ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(drow + (c >> 2) * BLK + (((cc + 1) ^ (r & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
    };
#pragma unroll 1
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      // scales are loaded two tiles ahead, table entries three
      const int tr = u.k0 * kTile + r;
      auto scale_of = [&](const float* scales, int64_t row) -> float {
        return kTok && row >= 0 ? __ldg(scales + row) : 0.0f;
      };
      Entry e0 = tok_entry(tr), e1 = tok_entry(tr + kTile), next_e = tok_entry(tr + 2 * kTile);
      int64_t row1 = row_of(tr, e0), row2 = row_of(tr + kTile, e1);
      float ks1 = scale_of(p.k_scales, row1), vs1 = scale_of(p.v_scales, row1);
      float ks2 = scale_of(p.k_scales, row2), vs2 = scale_of(p.v_scales, row2);
#pragma unroll 1
      for (int i = 0; i < tiles && ok; ++i) {
        const uint32_t k = g + i, rs = k % kRS, st = k % kKS, sv = k % kVS;
        const int t = tr + i * kTile;
        const int64_t row = row1;
        float ks = ks1, vs = vs1;
        row1 = row2;
        ks1 = ks2;
        vs1 = vs2;
        row2 = row_of(t + 2 * kTile, next_e);
        ks2 = scale_of(p.k_scales, row2);
        vs2 = scale_of(p.v_scales, row2);
        next_e = tok_entry(t + 3 * kTile);
        const bool node = t >= u.s.prefix;
        if (!(ok = wait(&rfull[rs], k / kRS))) break;
        const uint8_t* raw = smem + L::R0 + rs * 2 * L::RAW;
#pragma unroll 1
        for (int v = 0; v < 2; ++v) {  // K, then V (once PV of tile k - 2 is done, and its scales are read)
          if (!(ok = v == 0 ? wait(&kempty[st], k / kKS + 1) : wait(&vempty[sv], k / kVS + 1))) break;
          convert(raw + v * L::RAW, smem + (v == 0 ? L::K0 + st * TILE : L::V0 + sv * TILE), row >= 0);
          if (v == 0) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&kfull[st]);
          }
        }
        if (!ok) break;
        bool sick = false;
        if (std::is_same<CT, fp8>::value && node && row >= 0)
          sick = clear_sick<0x7c00u>(smem + L::V0 + sv * TILE + r * 128, kD * 2);
        if constexpr (kTok) {
          // P takes the token's V scale times 2^-vexp: a power of two that follows the largest
          // scale of a tile, moved only when that grows past it or falls 4 binades below. Where the
          // smallest lies far below the largest, the rows are told to take a unit of their own.
          if (node && !isfinite(vs)) {
            vs = 0.0f;
            sick = true;
          }
          const uint32_t ex = (__float_as_uint(vs) >> 23) & 255u;  // the scale's exponent
          const bool counts = ex != 0u && ex != 255u;
          const uint32_t wm = __reduce_max_sync(0xffffffffu, counts ? ex : 0u) |
                              __reduce_min_sync(0xffffffffu, counts ? ex : 255u) << 8;
          volatile uint32_t* mx = vmax_s + 4 * (k & 1);  // two sets: the other one may still be read
          if (lane == 0) {
            mx[warp - 12] = wm;
            mbar_arrive(cbar);
          }
          __syncwarp();
          if (!(ok = wait(cbar, k))) break;  // (bounded as every wait: another converter may have given up)
          int top = 0, low = 255;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = mx[j];
            top = max(top, (int)(x & 255u));
            low = min(low, (int)(x >> 8));
          }
          if (top > 0) {
            const int e = min(top - 127, 126);
            if (e > vexp || e < vexp - 4) vexp = e;
          }
          float* out = scales_s + sv * 2 * kTile;
          out[r] = ks;
          out[kTile + r] = vs * pow2f(-vexp);
          if (r == 0) vexp_s[sv] = 2 * vexp + (top > low + kWide);
        }
        if (sick) sick_s[unit % kSickSlots] = (int)unit + 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&vfull[sv]);
          mbar_arrive(&rempty[rs]);
        }
      }
      g += tiles;
      ++unit;
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
  if (*abort_flag) give_up<kRows, kTile, L::kThreads, QT>(p, reinterpret_cast<long long*>(smem + L::K0));
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {  // resolved once (thread-safe static initialisation)
  static const EncodeTiledFn fn = []() -> EncodeTiledFn {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(f);
    return nullptr;
  }();
  return fn;
}

template <typename QT, typename CT, bool kTok, int kD>
int launch(const Params& p, int cache_dtype, int ctas, cudaStream_t stream) {
  constexpr bool kByte = sizeof(CT) == 1;
  using L = Layout<kByte, kTok, kD>;
  // rows of the map = slots of the cache, each the kv heads' values; boxes of 128 bytes (8-bit
  // rows of 64: 64 bytes) x one page (or 128 tokens of it)
  const cuuint64_t dims[2] = {(cuuint64_t)p.num_kv_heads * kD, (cuuint64_t)p.num_blocks * (cuuint64_t)p.block_size};
  const cuuint64_t strides[1] = {(cuuint64_t)p.num_kv_heads * kD * sizeof(CT)};
  const cuuint32_t box[2] = {kByte ? (cuuint32_t)kD : 64u, (cuuint32_t)(p.block_size < kTile ? p.block_size : kTile)};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dt = kByte ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                       : (cache_dtype == MKV_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  // L2 fetches no more than a kv head's row of a token: with 256-byte fetches of 128-byte rows half of
  // what came was the next head's, gone before its turn (1.22 GB read for 0.81 GB of e4m3 pages)
  const CUtensorMapL2promotion promote = kD * sizeof(CT) >= 256   ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                         : kD * sizeof(CT) >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                                                  : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const CUresult r = encode_fn()(&maps[i], dt, 2, const_cast<uint8_t*>(i ? p.v_cache : p.k_cache), dims, strides, box,
                                   estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   kByte && kD == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                   promote, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(MKV_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  }
  const int st = ensure_dynamic_smem((const void*)paged_tree_tc_kernel<QT, CT, kTok, kD>, L::BYTES,
                                     "cudaFuncSetAttribute(paged_tree_tc smem)");
  if (st != MKV_OK) return st;
  paged_tree_tc_kernel<QT, CT, kTok, kD><<<ctas, L::kThreads, L::BYTES, stream>>>(p, maps[0], maps[1]);
  return cuda_status(cudaGetLastError(), "paged_tree_tc launch");
}

template <typename QT, int kD>
int launch_for(const Params& p, int cache_dtype, int ctas, cudaStream_t stream) {
  if (cache_dtype == MKV_DTYPE_FP8_E4M3)
    return p.k_scales ? launch<QT, fp8, true, kD>(p, cache_dtype, ctas, stream)
                      : launch<QT, fp8, false, kD>(p, cache_dtype, ctas, stream);
  if (cache_dtype == MKV_DTYPE_INT8) return launch<QT, int8_t, true, kD>(p, cache_dtype, ctas, stream);
  return launch<QT, QT, false, kD>(p, cache_dtype, ctas, stream);
}

}  // namespace

bool tc_supported(const Params& p, int q_dtype, int cache_dtype) {
  if ((p.head_dim != 64 && p.head_dim != 128) || (q_dtype != MKV_DTYPE_BF16 && q_dtype != MKV_DTYPE_F16)) return false;
  if (p.block_size < 8 || (p.block_size & (p.block_size - 1)) != 0) return false;
  if (p.num_blocks <= 0 || p.num_blocks * p.block_size > 0x7fffffffll) return false;  // TMA coordinates
  // 16-byte loads of query rows and stores of output rows
  if (((uintptr_t)p.q | (uintptr_t)p.out) & 15) return false;
  if (((p.q_st | p.q_sh | p.o_st | p.o_sh) & 7) != 0) return false;
  (void)cache_dtype;
  return encode_fn() != nullptr;
}

int launch_tc(const Params& p, int q_dtype, int cache_dtype, int ctas, cudaStream_t stream) {
  if (p.head_dim == 64)
    return q_dtype == MKV_DTYPE_BF16 ? launch_for<bf16, 64>(p, cache_dtype, ctas, stream)
                                     : launch_for<f16, 64>(p, cache_dtype, ctas, stream);
  return q_dtype == MKV_DTYPE_BF16 ? launch_for<bf16, 128>(p, cache_dtype, ctas, stream)
                                   : launch_for<f16, 128>(p, cache_dtype, ctas, stream);
}

}  // namespace tree
}  // namespace mkv
