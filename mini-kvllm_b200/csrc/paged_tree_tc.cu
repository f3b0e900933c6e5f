// Tree attention on the 5th-generation tensor cores: 16-bit queries, head_dim 128, pages of
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
//   warps 4-11  softmax of stream 0 (4-7) and 1 (8-11); they stage Q and write the output
//   warps 12-15 8-bit caches: converters of the raw tiles to f16 (exact) for the MMAs
// (warps 2 and 3 fill the first warpgroup, which gives registers to the softmax ones).
// K/V bytes are read once per unit of 128 rows; with fewer rows the tensor core's work is
// padded, which costs nothing while the tile's bytes take longer to arrive (bf16: 64 KB a
// tile, 1.5 us of an SM's share of HBM; its two products 0.55 us).
//
// What a row must not see: scores of hidden tokens are replaced by -inf before the maximum.
// Values meet P = 0 there, and 0 x inf is NaN, so rows of V that do not exist (past the
// context, missing pages) are zeroed in shared memory, and a tree's own rows, which some see
// and others do not, are searched for infinities and NaN: those are zeroed too, and added in
// at the end to the rows that see them.
//
// Every wait is bounded (sm100::kWaitCycles); a role that gives up raises the abort flag, the
// others stop, loads and MMAs in flight are waited for and TMEM is freed.
#include <cuda.h>

#include <type_traits>

#include "paged_tree.cuh"
#include "sm100.cuh"

namespace mkv {
namespace tree {
namespace {
using namespace sm100;

constexpr int kRows = kTcRows, kTile = 128, kD = 128;
constexpr int BLK = 128 * 128;   // 128 rows x 128 bytes
constexpr int TILE = 2 * BLK;    // a 16-bit tile: two halves of 64 columns
constexpr uint32_t kTmemCols = 512, kOCol = 256;
constexpr int kSickSlots = 4;

// kByte: 8-bit cache; kTok: with per-(token, head) scales.
template <bool kByte, bool kTok>
struct Layout {
  static constexpr int kThreads = kByte ? 512 : 384;
  // registers per thread after the split, of the launch's 512 x 128 or 384 x 168
  static constexpr int kRegsSoftmax = kByte ? 168 : 200, kRegsOther = kByte ? 88 : 104;
  static_assert(kByte ? 2 * kRegsSoftmax + 2 * kRegsOther <= 4 * 128 : 2 * kRegsSoftmax + kRegsOther <= 3 * 168,
                "more registers than the launch has");
  static constexpr int kKS = kByte ? 2 : 3;  // 16-bit K and V tiles
  static constexpr int kVS = 2;
  static constexpr int kRS = kByte ? 2 : 0;  // raw 8-bit tiles (K and V)
  static constexpr int Q0 = 0;
  static constexpr int K0 = Q0 + TILE;
  static constexpr int V0 = K0 + kKS * TILE;
  static constexpr int R0 = V0 + kVS * TILE;
  static constexpr int SC0 = R0 + kRS * 2 * BLK;             // [V stage][K scale, V factor][128]
  static constexpr int BAR0 = SC0 + (kTok ? kVS * 2 * kTile * 4 : 0);
  static constexpr int NBAR = 2 * kKS + 2 * kVS + 2 * kRS + 1 + 2 + 2 + 1 + 2 + 1;
  static constexpr int MISC0 = BAR0 + NBAR * 8;              // tmem base, abort, sick[4], exponents[2]
  static constexpr int BYTES = MISC0 + 64;
  static_assert(BYTES <= 232448, "shared memory per CTA");
  static_assert(kBeginWords(kThreads) * 8 <= TILE, "the schedule's scratch lies in the first K stage");
};

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

// Clears the infinities and NaN of a pair of 16-bit values (kExp: the type's exponent bits);
// true when there were any.
__device__ __forceinline__ bool clear_sick(uint32_t& w, uint32_t exp) {
  bool sick = false;
  if ((w & exp) == exp) {
    w &= 0xffff0000u;
    sick = true;
  }
  if ((w >> 16 & exp) == exp) {
    w &= 0x0000ffffu;
    sick = true;
  }
  return sick;
}

template <int N> __device__ __forceinline__ void regs_take() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_give() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float pow2f(int e) {  // 2^e, -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

template <typename QT, typename CT, bool kTok>
__global__ void __launch_bounds__((Layout<sizeof(CT) == 1, kTok>::kThreads), 1)
paged_tree_tc_kernel(const Params p, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap) {
  constexpr bool kByte = sizeof(CT) == 1;
  using L = Layout<kByte, kTok>;
  using MT = typename std::conditional<kByte, f16, QT>::type;  // operands of the MMAs
  // f16 weights: 2^6 above the reference, so that they stay normal down to 2^-20 of the
  // largest; with the lazy reference (2^8) and a scale factor below 2 they end below 2^15.
  constexpr float kBias = std::is_same<MT, f16>::value ? 6.0f : 0.0f;
  constexpr int kKS = L::kKS, kVS = L::kVS, kRS = kByte ? L::kRS : 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::BAR0);
  uint64_t* kempty = kfull + kKS;
  uint64_t* vfull = kempty + kKS;
  uint64_t* vempty = vfull + kVS;
  uint64_t* rfull = vempty + kVS;
  uint64_t* rempty = rfull + L::kRS;
  uint64_t* qfull = rempty + L::kRS;
  uint64_t* sfull = qfull + 1;
  uint64_t* pfull = sfull + 2;
  uint64_t* ofull = pfull + 2;
  uint64_t* xbar = ofull + 1;
  uint64_t* drain = xbar + 2;
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(smem + L::MISC0);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC0 + 4);
  volatile int* sick_s = reinterpret_cast<volatile int*>(smem + L::MISC0 + 8);
  volatile int* vexp_s = reinterpret_cast<volatile int*>(smem + L::MISC0 + 8 + 4 * kSickSlots);
  float* scales_s = reinterpret_cast<float*>(smem + L::SC0);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Walk walk;
  if (!begin<kRows, kTile, L::kThreads>(p, blockIdx.x, gridDim.x, reinterpret_cast<long long*>(smem + L::K0), walk))
    return;
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
    mbar_init(qfull, 8);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sfull[b], 1);
      mbar_init(&pfull[b], 4);
      mbar_init(&xbar[b], 8);
    }
    mbar_init(ofull, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    for (int i = 0; i < kSickSlots; ++i) sick_s[i] = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_base_s, kTmemCols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_base_s;
  // a tile is loaded in segments of one page (or of kTile tokens of a larger page)
  const int seg_rows = p.block_size < kTile ? p.block_size : kTile;
  const int nseg = kTile / seg_rows;
  auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {  // warp-uniform
    return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag));
  };
  // page of segment `lane` of tile t, -1 where it is missing or past the context
  auto seg_page_of = [&](const Unit& u, int t) -> int64_t {
    const int ts = t * kTile + lane * seg_rows;
    return (lane < nseg && ts < u.s.len) ? load_page(p, u.b, ts / p.block_size) : -1;
  };
  if (warp >= 4 && warp < 12) regs_take<L::kRegsSoftmax>();
  else regs_give<L::kRegsOther>();
  Unit u;
  uint32_t g = 0;     // tiles of this CTA before the unit's
  uint32_t unit = 0;  // units before this one
  bool ok = true;

  if (warp == 0) {
    // ================================================================ producer
    if (lane == 0) {
      tma_prefetch_map(&kmap);
      tma_prefetch_map(&vmap);
    }
    uint32_t nk = 0, nv = 0;  // K and V tiles issued (8-bit: nk counts both)
    // loads the rows of tile t that exist; the rest of the stage keeps what it held
    auto load = [&](const CUtensorMap* map, int t, int64_t page, uint32_t dst, uint64_t* bar) {
      for (int sgi = 0; sgi < nseg; ++sgi) {
        const int64_t pg = __shfl_sync(0xffffffffu, page, sgi);
        if (lane == 0 && pg >= 0) {
          const int y = (int)(pg * p.block_size) + ((t * kTile + sgi * seg_rows) & (p.block_size - 1));
          if constexpr (kByte) {
            tma_load_2d(dst + sgi * seg_rows * 128, map, u.kvh * kD, y, bar);
          } else {
            tma_load_2d(dst + sgi * seg_rows * 128, map, u.kvh * kD, y, bar);
            tma_load_2d(dst + BLK + sgi * seg_rows * 128, map, u.kvh * kD + 64, y, bar);
          }
        }
      }
      __syncwarp();
    };
    auto seg_bytes = [&](int64_t page) -> uint32_t {  // of one 8-bit tile or one half of a 16-bit one
      return (uint32_t)__popc(__ballot_sync(0xffffffffu, page >= 0)) * seg_rows * 128u;
    };
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      int64_t page_v = -1;
      for (int i = 0; i <= tiles && ok; ++i) {
        const int64_t page_k = i < tiles ? seg_page_of(u, u.k0 + i) : -1;
        if constexpr (kByte) {
          if (i == tiles) break;
          const uint32_t st = nk % kRS;
          if (!(ok = wait(&rempty[st], nk / kRS + 1))) break;
          const uint32_t bytes = 2 * seg_bytes(page_k);
          if (lane == 0) mbar_arrive_expect_tx(&rfull[st], bytes);
          __syncwarp();
          const uint32_t dst = smem_u32(smem + L::R0 + st * 2 * BLK);
          load(&kmap, u.k0 + i, page_k, dst, &rfull[st]);
          load(&vmap, u.k0 + i, page_k, dst + BLK, &rfull[st]);
          ++nk;
        } else {  // K one tile ahead of V, the order in which the products take them
          if (i < tiles) {
            const uint32_t st = nk % kKS;
            if (!(ok = wait(&kempty[st], nk / kKS + 1))) break;
            const uint32_t bytes = 2 * seg_bytes(page_k);
            if (lane == 0) mbar_arrive_expect_tx(&kfull[st], bytes);
            __syncwarp();
            load(&kmap, u.k0 + i, page_k, smem_u32(smem + L::K0 + st * TILE), &kfull[st]);
            ++nk;
          }
          if (i > 0) {
            const uint32_t st = nv % kVS;
            if (!(ok = wait(&vempty[st], nv / kVS + 1))) break;
            const uint32_t bytes = 2 * seg_bytes(page_v);
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
    if (lane == 0 && *abort_flag) {  // loads in flight land before the CTA exits
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
      if (lane == 0) {
        const uint32_t qaddr = smem_u32(smem + L::Q0), kaddr = smem_u32(smem + L::K0 + st * TILE);
#pragma unroll
        for (int c = 0; c < kD / 16; ++c) {  // 16 head_dim columns per MMA
          const uint32_t off = (c >> 2) * BLK + (c & 3) * 32;
          mma_f16(tmem + (i & 1) * kTile, smem_desc(qaddr + off, 16, 1024, kLayoutSw128),
                  smem_desc(kaddr + off, 16, 1024, kLayoutSw128), kIdQK, c > 0 ? 1u : 0u);
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
      if (lane == 0) {
        const uint32_t vaddr = smem_u32(smem + L::V0 + st * TILE);
#pragma unroll
        for (int c = 0; c < kTile / 16; ++c)  // 16 tokens per MMA: 8 columns of P
          mma_f16_ts(tmem + kOCol + (i & 1) * kD, tmem + (i & 1) * kTile + 8 * c,
                     smem_desc(vaddr + c * 2048, BLK, 1024, kLayoutSw128), kIdPV, (i > 1 || c > 0) ? 1u : 0u);
        mma_commit(&vempty[st]);
      }
      __syncwarp();
      return true;
    };
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      ok = wait(qfull, unit) && qk(0) && (tiles < 2 || qk(1));
      // QK(i + 2) is issued after PV(i), which reads the P that it overwrites; MMAs run in
      // the order of issue, so its S being full also says that PV(i) is done
      for (int i = 0; i < tiles && ok; ++i) ok = pv(i) && (i + 2 >= tiles || qk(i + 2));
      if (ok && lane == 0) mma_commit(ofull);
      __syncwarp();
      g += tiles;
      ++unit;
    }
    if (!ok) *abort_flag = 1;
    if (lane == 0) {  // every MMA done before TMEM is freed
      mma_commit(drain);
      mbar_wait(drain, 0, nullptr);
    }
    __syncwarp();
  } else if (warp >= 4 && warp < 12) {
    // ================================================================ softmax
    const int stream = (warp - 4) >> 2;       // also the half of the columns staged and written
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
    // the scale is made positive (a negative one turns Q around) and not 0, so that a masked
    // -inf stays one
    const bool flip = sc0 < 0.0f;
    sc0 = fabsf(sc0);
    if (sc0 < 1e-30f) sc0 = 1e-30f;
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      const int R = u.mt * kRows + rt, rows_left = u.s.nodes * p.group - u.mt * kRows;
      const bool live = rt < rows_left;
      const bool warp_live = 32 * (warp & 3) < rows_left;
      const int node = live ? R / p.group : 0;
      const int64_t qrow = u.s.q0 + node;
      const int head = u.kvh * p.group + (live ? R - node * p.group : 0);
      const uint64_t* mask_row = p.mask + qrow * p.mask_st;
      float sc = sc0;
      // ---- this thread's half of the row of Q (128-byte swizzle)
      {
        const QT* src = reinterpret_cast<const QT*>(p.q) + qrow * p.q_st + (int64_t)head * p.q_sh;
        uint8_t* dst = smem + L::Q0 + stream * BLK + rt * 128;
        float up = 1.0f;
        if constexpr (kByte && std::is_same<QT, bf16>::value) {
          // bf16 rows become f16 times a power of two that puts the largest value at 2^14: exact
          // down to 2^-28 of it
          float mx = 0.0f;
          if (live) {
#pragma unroll 4
            for (int c = 0; c < 16; ++c) {
              const uint4 v = *reinterpret_cast<const uint4*>(src + c * 8);
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                mx = fmax3(mx, fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u)));
            }
          }
          if (mx > 0.0f) {
            const int e = min(max(14 - ((int)(__float_as_uint(mx) >> 23) - 127), -100), 100);
            up = pow2f(e);
            sc *= pow2f(-e);
          }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (live) v = *reinterpret_cast<const uint4*>(src + stream * 64 + c * 8);
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (kByte && std::is_same<QT, bf16>::value)
              w[e] = pack2<f16>(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
            if (flip) w[e] ^= 0x80008000u;
          }
          *reinterpret_cast<uint4*>(dst + ((c ^ (rt & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);
      }
      float m = -INFINITY, l = 0.0f;  // reference (exp2 domain) and sum of this stream
      int vexp = 0;                   // O holds values times 2^-vexp (kTok)
      bool seen = false;
      int64_t page_next = seg_page_of(u, u.k0 + stream);
      for (int i = stream; i < tiles && ok; i += 2) {
        const int t0 = (u.k0 + i) * kTile;
        const uint32_t st = (g + i) % kVS, vph = (g + i) / kVS;
        const int64_t page = page_next;
        if (i + 2 < tiles) page_next = seg_page_of(u, u.k0 + i + 2);
        // ---- what the row sees: everything but in tiles with tree nodes, an end or a missing page
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
        const bool special = t0 + kTile > u.s.prefix || have != (nseg == 32 ? 0xffffffffu : (1u << nseg) - 1u);
        uint32_t mw[4];
        if (special) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mw[k] = visible32(u.s, mask_row, p.mask_words, t0 + 32 * k);
            uint32_t pm = 0;  // tokens 32k .. 32k + 31 that have a page
            for (int b = 0; b < 32; b += min(seg_rows, 32))
              if ((have >> ((32 * k + b) / seg_rows)) & 1u)
                pm |= (seg_rows >= 32 ? 0xffffffffu : (1u << seg_rows) - 1u) << b;
            mw[k] &= pm;
            seen |= mw[k] != 0u;
          }
        } else {
          seen = true;
        }
        if (!(ok = wait(&sfull[stream], ns))) break;  // also: PV of the stream's previous tile is done
        tc_fence_after_sync();
        const float* ksp = scales_s + st * 2 * kTile;
        float alpha = 1.0f;
        bool rescale = false;
        if constexpr (kTok) {  // the converters have written the tile's scales
          if (!(ok = wait(&vfull[st], vph))) break;
          const int e = vexp_s[st];
          if (e != vexp) {
            if (ns != 0) {
              alpha = exp2f((float)(vexp - e));
              rescale = true;
            }
            vexp = e;
          }
        }
        if (warp_live) {
          auto load_half = [&](int h, float (&v)[64]) {
            tmem_ld64(sa + 64 * h, v);
            if constexpr (kTok) {
#pragma unroll
              for (int e = 0; e < 64; e += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(ksp + 64 * h + e);
                v[e] *= k4.x;
                v[e + 1] *= k4.y;
                v[e + 2] *= k4.z;
                v[e + 3] *= k4.w;
              }
            }
            if (special) {
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (!((mw[2 * h + (e >> 5)] >> (e & 31)) & 1u)) v[e] = -INFINITY;
            }
          };
          // P = 2^(s sc - ref) of half h as 16-bit pairs, their sum, the raw maximum
          auto p_half = [&](int h, float ref, uint32_t (&w)[32], uint64_t (&acc)[2], float (&mx)[4]) {
            float v[64];
            load_half(h, v);
#pragma unroll
            for (int e = 0; e < 64; e += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) mx[k] = fmax3(mx[k], v[e + k], v[e + 4 + k]);
            const uint64_t sc2 = f2_pack(sc, sc), nref2 = f2_pack(-ref, -ref);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              float x0, x1;
              f2_unpack(f2_fma(f2_pack(v[2 * e], v[2 * e + 1]), sc2, nref2), x0, x1);
              float p0 = ex2_approx(x0), p1 = ex2_approx(x1);  // 0 where masked
              acc[e & 1] = f2_add(acc[e & 1], f2_pack(p0, p1));
              if constexpr (kTok) {
                const float2 f = *reinterpret_cast<const float2*>(ksp + kTile + 64 * h + 2 * e);
                p0 *= f.x;
                p1 *= f.y;
              }
              w[e] = pack2<MT>(p0, p1);
            }
          };
          uint32_t w0[32], w1[32];
          auto p_tile = [&](float ref, float& sum, float& mxr) {
            uint64_t acc[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            p_half(0, ref - kBias, w0, acc, mx);
            reg_fence32(w0);
            p_half(1, ref - kBias, w1, acc, mx);
            mxr = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
            float a, b, c, d;
            f2_unpack(acc[0], a, b);
            f2_unpack(acc[1], c, d);
            sum = (a + b) + (c + d);
          };
          float sum, mxr;
          bool need;
          // P against the reference as it is, together with the tile's maximum; again if a row's
          // maximum has grown by more than 2^8, or is its first
          const bool first = __any_sync(0xffffffffu, m == -INFINITY);
          if (first) {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              float v[64];
              load_half(h, v);
#pragma unroll
              for (int e = 0; e < 64; e += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = fmax3(mx[k], v[e + k], v[e + 4 + k]);
            }
            mxr = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
          } else {
            p_tile(m, sum, mxr);
          }
          const float mt = mxr * sc;
          need = mt > m + 8.0f;
          const float m_new = need ? mt : m;
          const float a2 = need ? exp2f(m - m_new) : 1.0f;  // 0 when m was -inf
          if (first || __any_sync(0xffffffffu, need)) {
            float unused;
            p_tile(m_new == -INFINITY ? 0.0f : m_new, sum, unused);
          }
          if (i > stream) {  // O holds something
            rescale |= __any_sync(0xffffffffu, need);
            alpha *= a2;
          }
          m = m_new;
          l = fmaf(l, a2, sum);
          tmem_st32(sa, w0);
          tmem_st32(sa + 32, w1);
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
#pragma unroll
            for (int k = 0; k < 16; ++k)
              *reinterpret_cast<uint4*>(vrow + (k >> 3) * BLK + (k & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          } else if (t >= u.s.prefix) {
            constexpr uint32_t kExp = std::is_same<QT, bf16>::value ? 0x7f80u : 0x7c00u;
            bool sick = false;
#pragma unroll 4
            for (int k = 0; k < 16; ++k) {
              uint4* at = reinterpret_cast<uint4*>(vrow + (k >> 3) * BLK + (k & 7) * 16);
              uint4 v = *at;
              bool here = clear_sick(v.x, kExp);
              here |= clear_sick(v.y, kExp);
              here |= clear_sick(v.z, kExp);
              here |= clear_sick(v.w, kExp);
              if (here) *at = v;
              sick |= here;
            }
            if (sick) sick_s[unit % kSickSlots] = (int)unit + 1;
          }
          fence_proxy_async_smem();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[stream]);
        ++ns;
      }
      // ---- the unit's end: both streams' references and sums change hands in S (free now)
      if (ok) ok = wait(ofull, unit);
      if (!ok) break;
      tc_fence_after_sync();
      tmem_st4(sa, m, l, (float)vexp, seen ? 1.0f : 0.0f);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&xbar[0]);
      if (!(ok = wait(&xbar[0], unit))) break;
      tc_fence_after_sync();
      if (warp_live) {
        float x[4];
        tmem_ld4(tmem + lane_base + (stream ^ 1) * kTile, x);
        const bool both = tiles > 1;
        const float M = both ? fmaxf(m, x[0]) : (stream == 0 ? m : x[0]);
        const float base = M == -INFINITY ? 0.0f : M;
        const float am = exp2f(m - base), ax = exp2f(x[0] - base);
        // (a stream without a tile has m = -inf and l = 0)
        const float lm = stream == 0 || both ? am * l : 0.0f, lx = stream == 1 || both ? ax * x[1] : 0.0f;
        float Ls = lm + lx;
        const bool any = seen || x[3] != 0.0f;
        const float a0 = vs0 * (stream == 0 ? am * exp2f((float)vexp) : ax * exp2f(x[2]));
        const float a1 = vs0 * (stream == 1 ? am * exp2f((float)vexp) : ax * exp2f(x[2]));
        const int slot = slot_of(u, blockIdx.x);
        float inv = 1.0f;
        if (slot < 0) inv = Ls == 0.0f ? (any ? NAN : 0.0f) : 1.0f / Ls;
        QT* dst = reinterpret_cast<QT*>(p.out) + qrow * p.o_st + (int64_t)head * p.o_sh + stream * 64;
        float* part = p.part_acc + ((int64_t)(slot < 0 ? 0 : slot) * kRows + rt) * kD + stream * 64;
        const bool sick = sick_s[unit % kSickSlots] == (int)unit + 1;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v[16];
          tmem_ld16(oa + stream * 64 + 16 * c, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= a0;
          if (both) {
            float y[16];
            tmem_ld16(oa + kD + stream * 64 + 16 * c, y);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = fmaf(y[e], a1, v[e]);
          }
          if (sick && live) {  // infinities and NaN of the nodes that the row sees
#pragma unroll 1
            for (int t = max(u.s.prefix, u.k0 * kTile); t < min(u.s.len, u.k1 * kTile); ++t) {
              const int64_t page = load_page(p, u.b, t / p.block_size);
              if (page < 0 || !(visible32(u.s, mask_row, p.mask_words, t) & 1u)) continue;
              const int64_t row = (page * p.block_size + (t & (p.block_size - 1))) * p.num_kv_heads + u.kvh;
              const CT* vr = reinterpret_cast<const CT*>(p.v_cache) + row * kD + stream * 64 + 16 * c;
              const float f = kTok ? __ldg(p.v_scales + row) : 1.0f;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float x2 = to_f32(vr[e]) * f;
                if (!isfinite(x2)) v[e] += x2;
              }
            }
          }
          if (!live) continue;
          if (slot < 0) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) w[e >> 1] = pack2<QT>(v[e] * inv, v[e + 1] * inv);
            *reinterpret_cast<uint4*>(dst + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(dst + 16 * c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(part + 16 * c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
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
    auto row_of = [&](int t) -> int64_t {  // (page, row, head) index of token t, -1
      if (t >= u.s.len) return -1;
      const int64_t page = load_page(p, u.b, t / p.block_size);
      return page < 0 ? -1 : (page * p.block_size + (t & (p.block_size - 1))) * p.num_kv_heads + u.kvh;
    };
    auto convert = [&](const uint8_t* src, uint8_t* dst, bool valid, bool node) -> bool {
      bool sick = false;
      uint8_t* drow = dst + r * 128;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t h[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        if (valid) {
          to_f16x16<CT>(*reinterpret_cast<const uint4*>(src + r * 128 + ((c ^ (r & 7)) << 4)), h);
          if (node && std::is_same<CT, fp8>::value) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sick |= clear_sick(h[e], 0x7c00u);
          }
        }
        const int cc = (c & 3) * 2;  // columns 16c ..: half c / 4, chunks cc and cc + 1
        *reinterpret_cast<uint4*>(drow + (c >> 2) * BLK + ((cc ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(drow + (c >> 2) * BLK + (((cc + 1) ^ (r & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      return sick;
    };
    while (ok && next<kRows, kTile>(p, walk, u)) {
      const int tiles = u.k1 - u.k0;
      int64_t row_next = row_of(u.k0 * kTile + r);
      for (int i = 0; i < tiles && ok; ++i) {
        const uint32_t k = g + i, rs = k % kRS, st = k % kKS, sv = k % kVS;
        const int t = (u.k0 + i) * kTile + r;
        const int64_t row = row_next;
        float ks = 0.0f, vs = 0.0f;
        if (kTok && row >= 0) {
          ks = __ldg(p.k_scales + row);
          vs = __ldg(p.v_scales + row);
        }
        if (i + 1 < tiles) row_next = row_of(t + kTile);
        const bool node = t >= u.s.prefix;
        if (!(ok = wait(&rfull[rs], k / kRS) && wait(&kempty[st], k / kKS + 1))) break;
        const uint8_t* raw = smem + L::R0 + rs * 2 * BLK;
        convert(raw, smem + L::K0 + st * TILE, row >= 0, false);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[st]);
        if (!(ok = wait(&vempty[sv], k / kVS + 1))) break;  // PV of tile k - 2 is done, and its scales are read
        bool sick = convert(raw + BLK, smem + L::V0 + sv * TILE, row >= 0, node);
        if constexpr (kTok) {
          // P takes the token's V scale times 2^-vexp: a power of two that follows the largest
          // scale of a tile, moved only when that grows past it or falls 4 binades below
          if (node && !isfinite(vs)) {
            vs = 0.0f;
            sick = true;
          }
          float* mx = scales_s + sv * 2 * kTile;
          const float a = isfinite(vs) ? fabsf(vs) : 0.0f;
          const float wm = warp_max(a);
          // the four warps' maxima, in the K-scale slots they fill next
          if (lane == 0) mx[32 * (warp - 12)] = wm;
          asm volatile("bar.sync 1, 128;" ::: "memory");
          const float tm = fmaxf(fmaxf(mx[0], mx[32]), fmaxf(mx[64], mx[96]));
          if (tm > 0.0f) {
            const int e = min(max((int)(__float_as_uint(tm) >> 23) - 127, -100), 100);
            if (e > vexp || e < vexp - 4) vexp = e;
          }
          asm volatile("bar.sync 1, 128;" ::: "memory");
          mx[r] = ks;
          mx[kTile + r] = vs * pow2f(-vexp);
          if (r == 0) vexp_s[sv] = vexp;
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

template <typename QT, typename CT, bool kTok>
int launch(const Params& p, int cache_dtype, int ctas, cudaStream_t stream) {
  constexpr bool kByte = sizeof(CT) == 1;
  using L = Layout<kByte, kTok>;
  // rows of the map = slots of the cache, each the kv heads' values; boxes of 128 bytes x one
  // page (or 128 tokens of it)
  const cuuint64_t dims[2] = {(cuuint64_t)p.num_kv_heads * kD, (cuuint64_t)p.num_blocks * (cuuint64_t)p.block_size};
  const cuuint64_t strides[1] = {(cuuint64_t)p.num_kv_heads * kD * sizeof(CT)};
  const cuuint32_t box[2] = {kByte ? 128u : 64u, (cuuint32_t)(p.block_size < kTile ? p.block_size : kTile)};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dt = kByte ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                       : (cache_dtype == MKV_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const CUresult r = encode_fn()(&maps[i], dt, 2, const_cast<uint8_t*>(i ? p.v_cache : p.k_cache), dims, strides, box,
                                   estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(MKV_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  }
  const int st = ensure_dynamic_smem((const void*)paged_tree_tc_kernel<QT, CT, kTok>, L::BYTES,
                                     "cudaFuncSetAttribute(paged_tree_tc smem)");
  if (st != MKV_OK) return st;
  paged_tree_tc_kernel<QT, CT, kTok><<<ctas, L::kThreads, L::BYTES, stream>>>(p, maps[0], maps[1]);
  return cuda_status(cudaGetLastError(), "paged_tree_tc launch");
}

template <typename QT>
int launch_for(const Params& p, int cache_dtype, int ctas, cudaStream_t stream) {
  if (cache_dtype == MKV_DTYPE_FP8_E4M3)
    return p.k_scales ? launch<QT, fp8, true>(p, cache_dtype, ctas, stream)
                      : launch<QT, fp8, false>(p, cache_dtype, ctas, stream);
  if (cache_dtype == MKV_DTYPE_INT8) return launch<QT, int8_t, true>(p, cache_dtype, ctas, stream);
  return launch<QT, QT, false>(p, cache_dtype, ctas, stream);
}

}  // namespace

bool tc_supported(const Params& p, int q_dtype, int cache_dtype) {
  if (p.head_dim != kD || (q_dtype != MKV_DTYPE_BF16 && q_dtype != MKV_DTYPE_F16)) return false;
  if (p.block_size < 8 || (p.block_size & (p.block_size - 1)) != 0) return false;
  if (p.num_blocks <= 0 || p.num_blocks * p.block_size > 0x7fffffffll) return false;  // TMA coordinates
  // 16-byte loads of query rows and stores of output rows
  if (((uintptr_t)p.q | (uintptr_t)p.out) & 15) return false;
  if (((p.q_st | p.q_sh | p.o_st | p.o_sh) & 7) != 0) return false;
  (void)cache_dtype;
  return encode_fn() != nullptr;
}

int launch_tc(const Params& p, int q_dtype, int cache_dtype, int ctas, cudaStream_t stream) {
  return q_dtype == MKV_DTYPE_BF16 ? launch_for<bf16>(p, cache_dtype, ctas, stream)
                                   : launch_for<f16>(p, cache_dtype, ctas, stream);
}

}  // namespace tree
}  // namespace mkv
