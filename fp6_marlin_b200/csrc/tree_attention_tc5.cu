// Attention over a paged cache for more than 32 rows per head of keys, on tcgen05 (fewer rows, and what is computed: tree_attention.cu).
//
// A row tile of 128 rows is the M dimension: scores S (128 x 128 keys, two key tiles: a job) = Q K^T with both operands in shared memory,
// then O (128 x head_dim) += P V with the weights P as the operand in tensor memory, written over S in 16 bits, and V as it lies (keys
// in rows, so its operand is "transposed").  A thread owns a row: no exchange between threads for maxima and sums.  Two groups of four warps
// compute weights, so that the tensor cores work on the product and the next scores of one while the other computes.  More than 128 rows: a group
// for each of two row tiles, which share the keys in shared memory.  Up to 128 rows: the groups take the jobs in turn and their sums
// are joined at the end.  (Jobs of 64 keys with two score tiles per group: the MMAs of 64 columns take 77 cycles each in place of 64 for 128,
// and what is passed between the warps, about 1300 cycles a job, bound the kernel.)
//
// O is rescaled only where a row's maximum grows by more than a factor of 2^8: until then the weights are taken relative to the older
// maximum, which changes neither the result nor, in fp32 sums and 16-bit floating-point weights, its precision.
//
// 2 x 64 tokens, 64 heads over 8, up to 32768 cached, public calls one behind the other: 190 us, 724 TFLOP/s, 0.43 of what a library product reaches (replays of a graph: 160
// to 176).  A job takes a pair of row tiles about 4700 cycles, the
// tensor cores 2048 of them: a group's weights take 2400 (the maxima 290, then 128 exponentials at 1660 to 2000: 660 of other instructions and 1024 of the unit for
// special functions, which a single warp per quarter does not overlap), then it waits for its product and its next scores, because tensor memory holds one
// tile of scores per group beside the sums.  Measured and not kept: a fourth, an eighth or a sixteenth of the exponentials by a polynomial (+3, +1, 0 %),
// sums and exponents in pairs (0), exponentials of one chunk between the sums of the last (+5 %, with or without registers moved to these warps).  The copies take 4 %.
// 64 x 7 tokens, 64 heads over 8, up to 6144: 182 us, 4.5 TB/s, 0.69 of what a copy reaches (in a graph: 158 to 170).  Figures of both sides of a choice are of replays of a graph.
//
// A cache in 8 bits (kFp8; cache_fp8.cu): two more warps bring tiles as they are, with their tokens' powers of two, and the copying warps widen them in place to 16 bits, so all behind
// them is the same.  Exact, so results are those of the widened cache.  2 x 64 tokens as above: 190 us in replays of a graph (16 bits there: 156 to 176): issue slots 49 %, a group's weights and the widening
// of the next tiles on the same schedulers.  64 x 5 / 16 tokens, 64 heads over 8, up to 6144: 241 / 256 us in bf16, 195 / 222 in fp16 (a conversion less for each pair).  Measured and not kept: 4-byte
// copies of the exponents that the widening warps decode (215 for the first, 318 for 64 x 5), all of a thread's powers read before its first store (213 / 283).
#include <type_traits>

#include "../../include/fp6m.h"
#include "device_utils.cuh"
#include "gemm_params.h"
#include "host_common.h"
#include "tc5_common.cuh"
#include "tree_attention.cuh"

namespace fp6m {

namespace {

constexpr int kRowTile = 128;
constexpr int kMostTreeCtas = 192;       // one per multiprocessor
constexpr int kTreeThreads = 512;        // four warps that copy, one that issues MMAs, three idle (with a cache in 8 bits two of them bring tiles), twice four that compute weights
// See make_plan (a pair's unit takes about twice as long).  us with a slack of 8 / 32: 8 x 16 tokens, 32 heads over 8, up to 2000 cached, 32.3 / 25.9; one of eight over 1000, 32
// over 4, 19.0 / 15.9; pairs, 16 / 32: one of 64 over 2000, 64 over 8, 38.9 / 47.0.  At least 3 / 6 / 9 units: that one 40.3 / 38.9 / 39.9; one of
// eight over 8000, 32 over 4, 28.7 / 27.9 / 29.4; four of eight over up to 3000 24.4 / 26.0 / 25.6.
constexpr int kSlack = 32, kPairSlack = 16, kLeastUnits = 6;

template <int D_, bool PAIR_, bool FP8_ = false>
struct TreeCfg {
  static constexpr int D = D_;
  static constexpr bool kFp8 = FP8_;                         // the cache is E4M3 with a power of two for each token and head
  static constexpr bool kPair = PAIR_;                       // two row tiles of an item share its keys, a group each; else the groups share one row tile
  static constexpr int kTileBytes = kKeys * D * 2;           // keys or values of a tile
  static constexpr int kQBytes = kRowTile * D * 2;
  // Stages of keys and of values, a job each.  Values are used later than their keys.
  static constexpr int kKeyStages = 2 * 128 / D, kValueStages = (kPair ? 2 : 3) * 128 / D;
  static constexpr int kStageBytes = 2 * kTileBytes, kHalfBytes = 2 * kKeys * 128;     // [half of a row][128 keys][64 values]
  static constexpr int kExchange = kRowTile * 32 * 4;        // 32 columns of a group's sums
  static constexpr int kNumBars = 2 * kKeyStages + 2 * kValueStages + 2 + 2 + 2 + 2 + (kFp8 ? kKeyStages + kValueStages : 0);
  static constexpr int kK = 0, kQ = kKeyStages * kStageBytes, kV = kQ + (kPair ? 2 : 1) * kQBytes, kX = kV + kValueStages * kStageBytes;
  static constexpr int kStats = kX + kExchange;              // [128] maxima, [128] totals of the second group
  static constexpr int kPlaces = kStats + 2 * kRowTile * 4;  // [keys, values][2][64] addresses
  static constexpr int kPowers = kPlaces + 4 * kKeys * 8;    // [stages of keys, then of values][128] powers of two of a job's tokens (kFp8)
  static constexpr int kBars = kPowers + (kFp8 ? (kKeyStages + kValueStages) * 2 * kKeys * 4 : 0);
  static constexpr int kSmemBytes = kBars + kNumBars * 8 + (4 + 32) * 4 + 1024;
  static constexpr int kSlotFloats = kRowTile * (D + 2) + 4; // a partial: sums [4 columns][row], maxima, totals, whether odd values were met
  static_assert(kSmemBytes <= 232448, "shared memory");
};
// Contributors of a group, see Joining.  Eight tokens over 8000, 32 heads over 4 (37 contributors): 66 us with all of them one after the other, 30 in two steps;
// four sequences of eight, up to 3000 (nine): 38 and 26, but with the planning of now 25.2 in one step of up to 12 and 27.0 in two.
__device__ __forceinline__ int join_step(int count) {
  if (count <= 12) return count;
  int step = 4;
  while (step * step < count) ++step;
  return step;
}
constexpr int kOddRing = 32;             // segments: more than the copies can be ahead of the sums

// operand with 128-byte swizzle whose 128-byte rows hold 64 values of K (keys and queries), or of N (`pitch`: from one 64 columns to the next)
__device__ __forceinline__ uint64_t rows_desc(uint32_t addr) { return wide_act_desc(addr); }
__device__ __forceinline__ uint64_t columns_desc(uint32_t addr, uint32_t pitch) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(pitch >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ float as_float(uint32_t v) { return __uint_as_float(v); }
// Four E4M3 values times a power of two, in 16 bits: exact where the type holds the result.  In fp16 one product a pair (the powers that it holds are those that it was written
// with).  of: the factor, from the exponent + 127; fp16 has those from kLeast to kMost.
template <class T> struct Widen;
template <> struct Widen<half> {
  static constexpr int kLeast = 127 - 24, kMost = 127 + 15;
  static __device__ __forceinline__ uint32_t of(int power) { return 0x10001u * __half_as_ushort(__float2half_rn(__uint_as_float((uint32_t)min(max(power, kLeast), kMost) << 23))); }
  static __device__ __forceinline__ void run(uint32_t four, uint32_t by, uint32_t& lo, uint32_t& hi) {
    lo = halves_of(four);
    hi = upper_halves_of(four);
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(by));
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(by));
  }
};
template <> struct Widen<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t of(int power) { return 0x10001u * ((uint32_t)min(max(power, 1), 254) << 7); }
  static __device__ __forceinline__ void run(uint32_t four, uint32_t by, uint32_t& lo, uint32_t& hi) {
    lo = halves_of(four);
    hi = upper_halves_of(four);
    const float2 p = __half22float2(*reinterpret_cast<half2*>(&lo)), q = __half22float2(*reinterpret_cast<half2*>(&hi));
    lo = Half16<__nv_bfloat16>::pack(p.x, p.y);
    hi = Half16<__nv_bfloat16>::pack(q.x, q.y);
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(lo) : "r"(by));
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(hi) : "r"(by));
  }
};

struct NoScales {};

// Scales: fp6m_cache_scales where the cache is in 8 bits.
template <class T, class C, class Scales>
__global__ void __launch_bounds__(kTreeThreads, 1) tree_attention_tc5_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ Scales scales, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  constexpr int D = C::D, SK = C::kKeyStages, SV = C::kValueStages;
  constexpr bool kPair = C::kPair;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = smem_u32(smem);
  const uint32_t full_k = base + C::kBars, empty_k = full_k + 8 * SK, full_v = empty_k + 8 * SK, empty_v = full_v + 8 * SV;
  const uint32_t q_free = empty_v + 8 * SV, scores = q_free + 16, weights = scores + 16, product = weights + 16, raw_k = product + 16, raw_v = raw_k + 8 * SK;
  volatile uint32_t* misc = reinterpret_cast<uint32_t*>(smem + C::kBars + C::kNumBars * 8);      // [0] TMEM base, [1] a page did not exist, or a power of two is none in fp16, [2, 3] last to arrive
  volatile uint32_t* odd_ring = misc + 4;                            // [segment]: infinities or NaN among its drafted values
  __shared__ Plan plan;
  const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31;
  const fp6m_tree_attention_args& a = p.a;

  if (tid == 0) {
    for (int s = 0; s < SK; ++s) {
      mbar_init(full_k + 8 * s, 128);        // the threads that copy, once for each of two key tiles: their copies have landed
      mbar_init(empty_k + 8 * s, 1);         // tcgen05.commit: the scores are computed
    }
    for (int s = 0; s < SV; ++s) {
      mbar_init(full_v + 8 * s, 128);
      mbar_init(empty_v + 8 * s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_free + 8 * i, 1);          // tcgen05.commit: an item's last scores are computed
      mbar_init(scores + 8 * i, 1);          // [group] tcgen05.commit
      mbar_init(weights + 8 * i, 4);         // [group] its warps have written the weights of a job
      mbar_init(product + 8 * i, 1);         // [group] tcgen05.commit: a segment's last weights are multiplied
    }
    if constexpr (C::kFp8)
      for (int i = 0; i < SK + SV; ++i) mbar_init(raw_k + 8 * i, 32);   // a warp that brings a job's tiles in 8 bits, and their powers of two
    mbar_fence_init();
    misc[1] = 0;
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(const_cast<uint32_t*>(misc))) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  launch_dependents();
  grid_dependency_wait();
  const int cta = blockIdx.x;
  if (warp == 0) make_plan(p, &plan, kLeastUnits, kPair ? kPairSlack : kSlack);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, misc[0], 0);
  const long long units = plan.units;
  const int ctas = plan.ctas;
  const bool works = cta < ctas;
  bool dead = false;
  // Up to 64 rows there is room for the queries of two items; a row tile is 128 rows all the same, what the others hold is nobody's.  The first group
  // has the rows in the first 64 lanes then and the second in the last, so that their warps share no quarter of the multiprocessor.
  const int q_rows = !kPair && p.rows <= 64 ? 64 : kRowTile, q_sets = !kPair && p.rows <= 64 ? 2 : 1;
  const uint32_t q_bytes = q_rows * D * 2;                           // of a row tile; halves of a row of 128 values lie q_rows * 128 bytes apart

  if (works) {
    Segments seg(p, plan);
    // score tiles [group][2] of 64 columns, then a tile of sums per group
    const uint32_t tmem_o = tmem + 256;
    if (warp < 4) {
      // ================================================================== copies: two warps the keys and queries, two the values
      const bool values = warp >= 2;
      const int me = tid & 63, chunk = me % (D / 8), row0 = me / (D / 8);
      constexpr int kRowsPerPass = 64 / (D / 8), kPasses = kKeys / kRowsPerPass;
      const uint32_t ring = base + (values ? C::kV : C::kK), full = values ? full_v : full_k, empty = values ? empty_v : empty_k;
      const T** places = reinterpret_cast<const T**>(smem + C::kPlaces) + (values ? 2 * kKeys : 0);
      const int bar_id = values ? 3 : 2;
      const CUtensorMap* map = values ? &vmap : &kmap;
      const int second = warp & 1, stages = values ? SV : SK;
      // Tiles of cached tokens come by tiled TMA, p.run tokens of a page at a time (0: the pages' size or the cache's layout does not allow it):
      // a warp those of the first 64 values, the other those of the second (heads of 64 values: every other run).  Other tiles, sixteen bytes a thread;
      // all tiles in that way took 2500 cycles of the copying warps each.
      // The first warp keeps the pages of 32 runs, a lane each, and those of the next 32 are on their way.
      const int tile_runs = p.run > 0 ? kKeys / p.run : 1, block_tiles = 32 / tile_runs, block_shift = 31 - __clz(block_tiles);
      constexpr int kWarpRuns = D == 128 ? 1 : 2;                    // a warp issues one of so many runs
      const uint32_t warp_bytes = p.run > 0 ? (D == 128 ? tile_runs : (tile_runs + 1 - second) / 2) * p.run * 128 : 0;
      Segments ahead = seg;
      auto pages_of = [&](int block) {
        const int j = (block * 32 + lane) * p.run;
        return page_of(p, ahead, j < ahead.length ? j : max(ahead.length - 1, 0));
      };
      int stage = 0, parity = 0, segment = 0;
      uint32_t phase = 1;                                            // of `empty`; the first round of stages is free
      // the queries of an item come with its first keys
      auto load_queries = [&] {
        const int set = segment % q_sets, turn = segment / q_sets;
        if (turn > 0) mbar_wait_bounded<50>(q_free + 8 * set, (turn - 1) & 1, p.status, dead);
        constexpr int kTiles = kPair ? 2 : 1;
        const int first_row = ahead.item % p.parts * kTiles * kRowTile;
        // (token and head are counted on: with a division for each row 256 of them took 20,000 cycles)
        const int r0 = first_row + row0, t0_q = r0 / p.group, step_t = kRowsPerPass / p.group, step_h = kRowsPerPass - step_t * p.group;
        const long long step = step_t * a.q_stride[1] + step_h * a.q_stride[2], wrap = a.q_stride[1] - p.group * a.q_stride[2];
        int h = r0 - t0_q * p.group;
        const T* src = static_cast<const T*>(a.q) + ahead.b * a.q_stride[0] + t0_q * a.q_stride[1] + (ahead.item / p.parts * p.group + h) * a.q_stride[2] + chunk * 8;
        const uint32_t q_to = base + C::kQ + (kPair ? 0 : set) * q_bytes + (chunk >> 3) * (q_rows * 128);
#pragma unroll 4
        for (int i = row0; i < kTiles * q_rows; i += kRowsPerPass) {
          const bool there = first_row + i < p.rows;
          copy16(q_to + (kPair ? i / kRowTile : 0) * q_bytes + (i & (q_rows - 1)) * 128 + (((chunk & 7) ^ (i & 7)) * 16), there ? src : static_cast<const T*>(a.q), there ? 16 : 0);
          src += step;
          h += step_h;
          if (h >= p.group) {
            h -= p.group;
            src += wrap;
          }
        }
      };
      if constexpr (C::kFp8) {
        // Cached tiles come as they are, E4M3, into the place of the 16-bit tile that they become (warps 5 and 6 bring them, see there); each thread takes sixteen values of a few tokens
        // and puts them back in 16 bits, times the token's power of two.  Heads of 128 values: a row lies where the first half of its 16-bit values goes, and both are one warp's; else
        // all threads have read a tile before any writes.  Tiles that TMA does not bring - the last ones of a sequence - are fetched here.
        const uint32_t raw = values ? raw_v : raw_k;
        const long long* cache_stride = values ? a.v_cache_stride : a.k_cache_stride;
        const uint8_t* cache = static_cast<const uint8_t*>(values ? a.v_cache : a.k_cache);
        const uint32_t* powers = reinterpret_cast<const uint32_t*>(smem + C::kPowers) + (values ? SK * 2 * kKeys : 0);
        constexpr int kNarrow = D / 16, kNarrowRows = 64 / kNarrow, kNarrowPasses = kKeys / kNarrowRows;    // 16-byte pieces of a row, rows of a pass
        const int narrow = me % kNarrow, narrow0 = me / kNarrow;
        phase = 0;                                                     // (here: of `raw`)
        while (__shfl_sync(0xffffffffu, (int)ahead.next(p), 0)) {
          const int t0 = __shfl_sync(0xffffffffu, ahead.t0, 0), t1 = __shfl_sync(0xffffffffu, ahead.t1, 0), length = __shfl_sync(0xffffffffu, ahead.length, 0);
          const int g = __shfl_sync(0xffffffffu, ahead.item / p.parts, 0);
          if (values) {
            if (me == 0) odd_ring[segment % kOddRing] = 0;
          } else {
            load_queries();
          }
#pragma unroll 1
          for (int tile = t0; tile < t1; tile += 2) {
            mbar_wait_bounded<20>(raw + 8 * stage, phase, p.status, dead);
            const uint32_t bar = full + 8 * stage;
#pragma unroll 1
            for (int odd_tile = 0; odd_tile < 2; ++odd_tile) {
              const uint32_t at = ring + stage * C::kStageBytes + odd_tile * (kKeys * 128);
              const int at_tile = tile + odd_tile;
              if (at_tile < t1) {
                const int cached = min(length - at_tile * kKeys, kKeys);
                const bool by_tma = p.run > 0 && cached == kKeys, apart = D == 128 && by_tma;
                if (!by_tma) {
                  // a thread works out where its token is
                  const uint8_t** narrow_places = reinterpret_cast<const uint8_t**>(places);
                  const int j = at_tile * kKeys + me, page = j < length ? page_of(p, ahead, j) : -1;
                  const int slot = j - (int)((unsigned long long)j * p.page_magic >> p.page_shift) * a.page_size;
                  narrow_places[me] = (unsigned)page < (unsigned)a.pages ? cache + page * cache_stride[0] + slot * cache_stride[1] + g * cache_stride[2] : nullptr;
                  named_bar_sync(bar_id, 64);
#pragma unroll 4
                  for (int i = 0; i < kNarrowPasses; ++i) {
                    const int row = narrow0 + i * kNarrowRows;
                    const uint8_t* src = narrow_places[row];
                    if (row < cached) copy16(at + row * D + narrow * 16, src ? src + narrow * 16 : static_cast<const uint8_t*>(a.q), src ? 16 : 0);
                  }
                  // drafted tokens as they are; zeros behind them
                  const long long* drafted_stride = values ? a.v_stride : a.k_stride;
                  for (int row = row0; row < kKeys; row += kRowsPerPass) {
                    const int t = at_tile * kKeys + row - length;
                    if (t < 0) continue;
                    const T* src = static_cast<const T*>(values ? a.v : a.k) + ahead.b * drafted_stride[0] + min(t, a.tokens - 1) * drafted_stride[1] + g * drafted_stride[2];
                    copy16(at + (chunk >> 3) * C::kHalfBytes + row * 128 + (((chunk & 7) ^ (row & 7)) * 16), src + chunk * 8, t < a.tokens ? 16 : 0);
                  }
                }
                if (!by_tma || (!values && tile == t0)) asm volatile("cp.async.wait_all;" ::: "memory");      // (the queries, too)
                if (!apart) named_bar_sync(bar_id, 64);
                uint32_t v[kNarrowPasses][4];
#pragma unroll
                for (int i = 0; i < kNarrowPasses; ++i) {
                  const uint4 w = lds128(at + (narrow0 + i * kNarrowRows) * D + narrow * 16);
                  v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
                }
                if (apart) __syncwarp();
                else named_bar_sync(bar_id, 64);
#pragma unroll
                for (int i = 0; i < kNarrowPasses; ++i) {
                  const int row = narrow0 + i * kNarrowRows;
                  const uint32_t by = powers[(stage * 2 + odd_tile) * kKeys + row];
                  uint32_t w[8];
#pragma unroll
                  for (int e = 0; e < 4; ++e) Widen<T>::run(v[i][e], by, w[2 * e], w[2 * e + 1]);
                  const uint32_t to = at + (2 * narrow >> 3) * C::kHalfBytes + row * 128;
                  if (row < cached) {
                    sts128(to + (((2 * narrow & 7) ^ (row & 7)) * 16), w);
                    sts128(to + (((2 * narrow & 7) + 1 ^ (row & 7)) * 16), w + 4);
                  }
                }
                if (values && cached < kKeys) {
                  // Infinities and NaN among the drafted values: a weight of zero must not meet them.  They are zero in the product, and added to the rows
                  // that see them at the end.
                  named_bar_sync(bar_id, 64);
                  bool odd = false;
                  if (me >= cached) {
                    for (int c = 0; c < D / 8; ++c) {
                      const uint32_t place = at + (c >> 3) * C::kHalfBytes + me * 128 + (((c & 7) ^ (me & 7)) * 16);
                      const uint4 w = lds128(place);
                      uint32_t x[4] = {w.x, w.y, w.z, w.w};
                      constexpr uint32_t E = Half16<T>::kExponent;
                      for (int e = 0; e < 4; ++e) {
                        if (!is_odd<T>(x[e])) continue;
                        odd = true;
                        if ((x[e] & E) == E) x[e] &= 0xffff0000u;
                        if ((x[e] >> 16 & E) == E) x[e] &= 0xffffu;
                        sts_u32(place + 4 * e, x[e]);
                      }
                    }
                  }
                  if (odd) odd_ring[segment % kOddRing] = 1;
                }
                // what was stored is seen by the MMAs, and by the copies that come into this place later
                fence_async_proxy();
              }
              mbar_arrive(bar);
            }
            if (++stage == stages) { stage = 0; phase ^= 1; }
          }
          ++segment;
        }
      } else {
      while (__shfl_sync(0xffffffffu, (int)ahead.next(p), 0)) {
        // What follows from the lengths is made uniform to the compiler (read from lane 0): copies whose operands it takes to differ between
        // lanes cost 150 cycles each to issue.
        const int t0 = __shfl_sync(0xffffffffu, ahead.t0, 0), t1 = __shfl_sync(0xffffffffu, ahead.t1, 0), length = __shfl_sync(0xffffffffu, ahead.length, 0);
        const int g = __shfl_sync(0xffffffffu, ahead.item / p.parts, 0);
        if (values) {
          if (me == 0) odd_ring[segment % kOddRing] = 0;
        } else {
          load_queries();
        }
        int pages = 0, pages_next = 0, slot = 0;
        if (p.run > 0) {
          pages = pages_of(t0 >> block_shift);
          pages_next = pages_of((t0 >> block_shift) + 1);
          slot = t0 * kKeys - (int)((unsigned long long)(t0 * kKeys) * p.page_magic >> p.page_shift) * a.page_size;
        }
#pragma unroll 1
        for (int tile = t0; tile < t1; ++tile) {
        const int odd_tile = (tile - t0) & 1;
        const uint32_t dst = ring + stage * C::kStageBytes + odd_tile * (kKeys * 128), bar = full + 8 * stage;
        const bool runs = p.run > 0 && (tile + 1) * kKeys <= length;
        bool missing = false;                                      // this thread has found a page that does not exist
        const bool drafted = values && (tile + 1) * kKeys > length;
        if (runs) {
          const int at = tile & (block_tiles - 1);
          if (at == 0 && tile != t0) {
            pages = pages_next;
            pages_next = pages_of((tile >> block_shift) + 1);
          }
          if (!odd_tile) mbar_wait_bounded<50>(empty + 8 * stage, phase, p.status, dead);
          if (elect_one()) mbar_expect_tx(bar, warp_bytes);
          __syncwarp();
#pragma unroll 1
          for (int i = 0; i < tile_runs; ++i) {
            int page = __shfl_sync(0xffffffffu, pages, at * tile_runs + i);
            if ((unsigned)page >= (unsigned)a.pages) {
              missing = true;
              page = a.pages;                                        // behind the last page the copy reads zeros
            }
            if (kWarpRuns == 1 || (i & 1) == second) {
              if (elect_one()) tma_load_run(dst + (D == 128 ? second : 0) * C::kHalfBytes + i * p.run * 128, map, D == 128 ? second * 64 : 0, g, slot, page, bar);
              __syncwarp();
            }
            slot += p.run;
            if (slot == a.page_size) slot = 0;
          }
        } else {
          const int j = tile * kKeys + me;
          const T* place = place_of<T>(p, ahead, g, j, page_of(p, ahead, j), values);
          missing = !place && j < length;
          places[parity * kKeys + me] = place;
          named_bar_sync(bar_id, 64);
          if (!odd_tile) mbar_wait_bounded<50>(empty + 8 * stage, phase, p.status, dead);
#pragma unroll 4
          for (int i = 0; i < kPasses; ++i) {
            const int row = row0 + i * kRowsPerPass;
            const T* src = places[parity * kKeys + row];
            copy16(dst + (chunk >> 3) * C::kHalfBytes + row * 128 + (((chunk & 7) ^ (row & 7)) * 16), src ? src + chunk * 8 : static_cast<const T*>(a.q), src ? 16 : 0);
          }
          parity ^= 1;
        }
        // The arrival of asynchronous copies does not order a thread's stores, a plain one does.
        missing = __any_sync(0xffffffffu, missing);
        if (missing) misc[1] = 1;
        if (!drafted && missing) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          mbar_arrive(bar);
        } else if (!drafted) {
          copies_arrive(bar);
        }
        if (drafted) {
          // Infinities and NaN among the drafted values: a weight of zero must not meet them.  They are zero in the product, and added to the rows
          // that see them at the end.
          asm volatile("cp.async.wait_all;" ::: "memory");
          named_bar_sync(bar_id, 64);
          const int j = tile * kKeys + me;
          bool odd = false;
          if (j >= length) {
            for (int c = 0; c < D / 8; ++c) {
              const uint32_t at = dst + (c >> 3) * C::kHalfBytes + me * 128 + (((c & 7) ^ (me & 7)) * 16);
              uint4 w = lds128(at);
              if (is_odd<T>(w.x) || is_odd<T>(w.y) || is_odd<T>(w.z) || is_odd<T>(w.w)) {
                odd = true;
                uint32_t v[4] = {w.x, w.y, w.z, w.w};
                constexpr uint32_t E = Half16<T>::kExponent;
                for (int e = 0; e < 4; ++e) {
                  if ((v[e] & E) == E) v[e] &= 0xffff0000u;
                  if ((v[e] >> 16 & E) == E) v[e] &= 0xffffu;
                  sts_u32(at + 4 * e, v[e]);
                }
              }
            }
          }
          if (odd) odd_ring[segment % kOddRing] = 1;
          mbar_arrive(bar);
        }
        if (!odd_tile && tile + 1 == t1) mbar_arrive(bar);           // for the second tile that the job does not have
        if ((odd_tile || tile + 1 == t1) && ++stage == stages) { stage = 0; phase ^= 1; }
        }
        ++segment;
      }
      }
    } else if (warp == 4) {
      // ================================================================== MMA issuer
      constexpr uint32_t kFormats = (1u << 4) | (Half16<T>::kMmaFormat << 7) | (Half16<T>::kMmaFormat << 10) | ((uint32_t)(kRowTile >> 4) << 24);
      const uint32_t sign = p.scale_log2 < 0.f ? 1u << 13 : 0u;      // the queries are negated
      const uint32_t idesc_s = kFormats | sign | ((uint32_t)(kKeys >> 3) << 17), idesc_s2 = kFormats | sign | ((uint32_t)(2 * kKeys >> 3) << 17);
      constexpr uint32_t idesc_o = kFormats | (1u << 16) | ((uint32_t)(D >> 3) << 17);         // values are N-major
      // What follows from the lengths is made uniform to the compiler (read from lane 0), so that MMAs are issued with uniform operands.
      struct Jobs {
        Segments seg;
        int left, plain, groups;                                     // key tiles of the segment that are left, of them those that TMA brings; groups
        int stage;
        uint32_t phase;
        __device__ __forceinline__ bool next(const TreeParams& p) {
          const bool lives = seg.next(p);
          left = __shfl_sync(0xffffffffu, lives ? seg.t1 - seg.t0 : 0, 0);
          plain = C::kFp8 ? left : p.run > 0 ? __shfl_sync(0xffffffffu, min(seg.t1, seg.length / kKeys) - seg.t0, 0) : 0;      // (widened tiles are fenced by who stores them)
          // of a pair of row tiles, the second may have no rows
          groups = __shfl_sync(0xffffffffu, kPair && seg.item % p.parts * 2 + 1 < p.row_tiles ? 2 : 1, 0);
          return left > 0;
        }
        // waits for the next stage; other copies than TMA's (the queries come with a segment's first) need a proxy fence, so that the MMAs that follow see them.  It stands here, behind the
        // barrier that counts the copies: in a thread that copies it would wait for all of that thread's copies in flight (measured: a tile per latency of memory, 7000
        // cycles, in place of four tiles on their way).
        __device__ __forceinline__ void wait(uint32_t full, bool other_copies, int* status, bool& dead) {
          mbar_wait_bounded<20>(full + 8 * stage, phase, status, dead);
          if (other_copies || plain < min(left, 2)) fence_async_proxy();
          tc_fence_after();
        }
        __device__ __forceinline__ bool advance(const TreeParams& p, int stages) {
          if (++stage == stages) { stage = 0; phase ^= 1; }
          left -= 2;
          plain -= 2;
          return left > 0 || next(p);
        }
      };
      Jobs front = {seg, 0, 0, 0, 0, 0}, back = front;               // of the scores, of the products
      bool front_lives = front.next(p), back_lives = back.next(p), fresh = true;       // fresh: a segment's first scores
      int segment = 0, scored = 0, multiplied = 0, part = 0;         // jobs; the group whose scores of the front job are next
      uint32_t weight_phase = 0, started = 0;                        // of both groups, a bit each; groups whose sums of the segment hold something
      // scores of the front job for group w; the job is done with the last group's
      auto issue_scores = [&](int w) {
        const int set = q_sets == 2 ? segment & 1 : 0;
        if (!kPair || w == 0) front.wait(full_k, fresh, p.status, dead);
        fresh = false;
        const uint64_t k_desc = rows_desc(base + C::kK + front.stage * C::kStageBytes), q_desc = rows_desc(base + C::kQ + (kPair ? w : set) * q_bytes - (q_sets == 2 && w == 1 ? 64 * 128 : 0));
        const uint32_t idesc = front.left > 1 ? idesc_s2 : idesc_s;
        const bool whole_job = !kPair || w + 1 == front.groups;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_smem(tmem + w * 128, q_desc + (i >> 2) * (q_rows * 128 >> 4) + (i & 3) * 2, k_desc + (i >> 2) * (C::kHalfBytes >> 4) + (i & 3) * 2, idesc, i);
          tc_commit(scores + 8 * w);
          if (whole_job) {
            tc_commit(empty_k + 8 * front.stage);
            if (front.left <= 2) tc_commit(q_free + 8 * set);
          }
        }
        __syncwarp();
        part = whole_job ? 0 : w + 1;
        if (whole_job) {
          ++scored;
          if (front.left <= 2) {
            ++segment;
            fresh = true;
          }
          front_lives = front.advance(p, SK);
        }
      };
      if constexpr (kPair) {
        if (front_lives) {                                           // (a range may hold nothing but the overhead of an item)
          do issue_scores(part); while (part);
        }
      } else {
        for (int i = 0; i < 2 && front_lives; ++i) issue_scores(scored & 1);
      }
      while (back_lives) {
        back.wait(full_v, false, p.status, dead);
        const uint64_t v_desc = columns_desc(base + C::kV + back.stage * C::kStageBytes, C::kHalfBytes);
        // the group's last job of the segment
        const bool last = kPair ? back.left <= 2 : back.left <= 4;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (kPair ? w >= back.groups : w != (multiplied & 1)) continue;
          mbar_wait_bounded<20>(weights + 8 * w, weight_phase >> w & 1, p.status, dead);
          weight_phase ^= 1u << w;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < 2 * kKeys / 16; ++i)
              if (i < kKeys / 16 || back.left > 1) mma_tmem(tmem_o + w * 128, tmem + w * 128 + i * 8, v_desc + i * (16 * 128 >> 4), idesc_o, i > 0 ? 1u : started >> w & 1);
            if (last) tc_commit(product + 8 * w);
            if (!kPair || w + 1 == back.groups) tc_commit(empty_v + 8 * back.stage);
          }
          __syncwarp();
          started |= 1u << w;
          // the group's next scores, over the weights that the product has read by then
          if (front_lives && (!kPair || part == w)) {
            if constexpr (kPair) {
              // (the front job is the one behind this: not that of the next turn)
              if (scored == multiplied + 1) issue_scores(w);
            } else {
              issue_scores(w);
            }
          }
        }
        if constexpr (kPair) {
          while (part) issue_scores(part);
        }
        ++multiplied;
        const bool segment_ends = back.left <= 2;
        back_lives = back.advance(p, SV);
        if (segment_ends) started = 0;
      }
    } else if (C::kFp8 && (warp == 5 || warp == 6)) {
      // ================================================================== tiles in 8 bits: a warp the keys, one the values
      if constexpr (C::kFp8) {
        const bool values = warp == 6;
        const uint32_t ring = base + (values ? C::kV : C::kK), empty = values ? empty_v : empty_k, raw = values ? raw_v : raw_k;
        const int stages = values ? SV : SK;
        const CUtensorMap* map = values ? &vmap : &kmap;
        const void* power_base = values ? scales.v_scales : scales.k_scales;
        const long long* power_stride = values ? scales.v_scales_stride : scales.k_scales_stride;
        const unsigned power_page = (unsigned)power_stride[0], power_slot = (unsigned)power_stride[1];
        uint32_t* powers = reinterpret_cast<uint32_t*>(smem + C::kPowers) + (values ? SK * 2 * kKeys : 0);
        // the pages of 32 runs, a lane each, and those of the next 32 are on their way; without runs each token's is looked up
        const int tile_runs = p.run > 0 ? kKeys / p.run : 1, block_tiles = 32 / tile_runs, block_shift = 31 - __clz(block_tiles), run_log2 = __ffs(max(p.run, 1)) - 1, step_slots = kKeys % a.page_size;
        auto pages_of = [&](int block) {
          const int j = (block * 32 + lane) * p.run;
          return j < seg.length ? page_of(p, seg, j) : -1;
        };
        int stage = 0;
        uint32_t phase = 1;                                            // of `empty`; the first round of stages is free
        while (__shfl_sync(0xffffffffu, (int)seg.next(p), 0)) {
          const int t0 = __shfl_sync(0xffffffffu, seg.t0, 0), t1 = __shfl_sync(0xffffffffu, seg.t1, 0), length = __shfl_sync(0xffffffffu, seg.length, 0);
          const int g = __shfl_sync(0xffffffffu, seg.item / p.parts, 0);
          const uint8_t* head_powers = static_cast<const uint8_t*>(power_base) + g * power_stride[2];
          int block = t0 >> block_shift, pages = 0, pages_next = 0, slot[2], power[2][2];
          if (p.run > 0) {
            pages = pages_of(block);
            pages_next = pages_of(block + 1);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int j = t0 * kKeys + 32 * i + lane;
            slot[i] = j - (int)((unsigned long long)j * p.page_magic >> p.page_shift) * a.page_size;
          }
          int first_slot = __shfl_sync(0xffffffffu, slot[0], 0);
          bool missing = false;
          // the exponents of a job's tokens; looked up while the job before is waited for
          auto look_up = [&](int tile) {
#pragma unroll
            for (int odd_tile = 0; odd_tile < 2; ++odd_tile) {
              const int at_tile = tile + odd_tile, of_block = at_tile >> block_shift == block ? pages : pages_next;
              power[odd_tile][0] = power[odd_tile][1] = 127;
              if (at_tile >= t1) continue;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int in = 32 * i + lane, j = at_tile * kKeys + in;
                const int page = p.run > 0 ? __shfl_sync(0xffffffffu, of_block, (at_tile & (block_tiles - 1)) * tile_runs + (in >> run_log2)) : j < length ? page_of(p, seg, j) : -1;
                if (j < length) {
                  const bool known = (unsigned)page < (unsigned)a.pages;
                  if (known) power[odd_tile][i] = head_powers[(unsigned long long)(unsigned)page * power_page + (unsigned long long)(unsigned)slot[i] * power_slot];
                  missing = missing || !known;
                }
                slot[i] += step_slots;
                if (slot[i] >= a.page_size) slot[i] -= a.page_size;
              }
            }
          };
          look_up(t0);
#pragma unroll 1
          for (int tile = t0; tile < t1; tile += 2) {
            mbar_wait_bounded<20>(empty + 8 * stage, phase, p.status, dead);
            const uint32_t bar = raw + 8 * stage;
#pragma unroll 1
            for (int at_tile = tile; at_tile < min(tile + 2, t1); ++at_tile) {
              if (p.run > 0 && at_tile >> block_shift != block) {
                ++block;
                pages = pages_next;
                pages_next = pages_of(block + 1);
              }
              if (p.run > 0 && (at_tile + 1) * kKeys <= length) {
                const uint32_t dst = ring + stage * C::kStageBytes + (at_tile - tile) * (kKeys * 128);
                const int in_block = at_tile & (block_tiles - 1);
                if (elect_one()) mbar_expect_tx(bar, kKeys * D);
                __syncwarp();
                auto bring = [&](auto runs) {
                  constexpr int R = decltype(runs)::value;
                  int of[R];
#pragma unroll
                  for (int r = 0; r < R; ++r) {
                    of[r] = __shfl_sync(0xffffffffu, pages, in_block * R + r);
                    if ((unsigned)of[r] >= (unsigned)a.pages) of[r] = a.pages;        // behind the last page the copy reads zeros
                  }
                  if (elect_one()) {
                    int from = first_slot;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                      tma_load_run(dst + r * (kKeys / R) * D, map, 0, g, from, of[r], bar);
                      from += kKeys / R;
                      if (from == a.page_size) from = 0;
                    }
                  }
                  __syncwarp();
                };
                if (tile_runs == 1) bring(std::integral_constant<int, 1>());
                else if (tile_runs == 2) bring(std::integral_constant<int, 2>());
                else if (tile_runs == 4) bring(std::integral_constant<int, 4>());
                else bring(std::integral_constant<int, 8>());
              }
              first_slot += step_slots;
              if (first_slot >= a.page_size) first_slot -= a.page_size;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int of = power[i >> 1][i & 1];
              powers[stage * 2 * kKeys + 32 * i + lane] = Widen<T>::of(of);
              // (reported alike; not where it is looked up, which would wait for it: 39 -> 57 us for 8 x 16 tokens over up to 2000)
              if constexpr (Half16<T>::kMmaFormat == 0) missing = missing || of < Widen<T>::kLeast || of > Widen<T>::kMost;
            }
            if (missing) misc[1] = 1;
            mbar_arrive(bar);
            if (++stage == stages) { stage = 0; phase ^= 1; }
            look_up(tile + 2);
          }
        }
      }
    } else if (warp >= 8) {
      // ================================================================== weights: thread = row
      const int group = (warp - 8) >> 2, quarter = warp & 3, first_lane = q_sets == 2 && group == 1 ? 64 : 0;
      const int row_in = quarter * 32 + lane - first_lane;           // negative: nobody's
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const uint32_t my_scores = tmem + lanes + group * 128, my_sums = tmem_o + lanes + group * 128;
      const float sl = fabsf(p.scale_log2);                          // its sign is in the scores
      float* stats = reinterpret_cast<float*>(smem + C::kStats);
      float4* exchange = reinterpret_cast<float4*>(smem + C::kX);
      int job = 0, n = 0, segment = -1, ended = 0;                   // jobs of this group, jobs of the CTA; segments that this group has jobs of
      while (seg.next(p)) {
        ++segment;
        const int g = seg.item / p.parts, row_tile = kPair ? seg.item % p.parts * 2 + group : seg.item % p.parts;
        const int row = row_tile * kRowTile + row_in;
        const bool warp_lives = quarter * 32 >= first_lane && row_tile * kRowTile + quarter * 32 - first_lane < p.rows;
        bool row_lives = row_in >= 0 && row < p.rows;
        const int t = row_lives ? row / p.group : 0, head = g * p.group + (row_lives ? row - t * p.group : 0);
        unsigned long long mask = row_lives ? mask_of(p, seg.b, t) : 0;
        float top = -INFINITY, total = 0.f;                          // the maximum that the weights are relative to
        bool any = false;                                            // the sums hold something
        bool rounds = false;                                         // scores are rounded before the maximum is taken from them
        const bool group_lives = !kPair || row_tile < p.row_tiles;
        for (int tile = seg.t0; tile < seg.t1; tile += 2, ++n) {
          if (!group_lives || (!kPair && (n & 1) != group)) continue;
          mbar_wait_bounded<20>(scores + 8 * group, job & 1, p.status, dead);
          tc_fence_after();
          if (warp_lives) {
            const int chunks = tile + 1 < seg.t1 ? 4 : 2;            // of 32 keys
            const int cached = seg.length - tile * kKeys;            // from the job's first key on
            // One answer for the warp: the copies run ahead and set the flag at any time, and the two bodies below hold warp-wide instructions.
            const bool hidden = __any_sync(0xffffffffu, misc[1] != 0);
            // The largest score, then the weights: scores are read twice, because 128 of them would not stay in registers.  `hides`: some of the job's keys are
            // not seen by every row.  (A branch for every 32 scores, for what is hidden or grows, cost 150 cycles each: the two cases are apart.)
            // A fused multiply-add leaves the rounding of the maximum, 2^-24 of it, in the exponent, and at 2^28 weights leave fp16's range: from 2^22 on (a quarter) scores are
            // rounded as it was, so that the largest has a weight of 1.  That is done with what is hidden: false, and there are no weights, where a job turns out to need it.
            // (A second copy of the exponentials in each case took 10 % longer for 64 x 5 tokens: it does not fit beside the rest of the code.)
            auto weigh = [&](auto hides) {
              constexpr bool kHides = decltype(hides)::value;
              // The row sees all cached keys, then those of its mask; the score of another is the lowest there is.
              uint32_t sees[4] = {~0u, ~0u, ~0u, ~0u};
              if constexpr (kHides) {
                const unsigned long long drafted = mask & (~0ull >> (64 - a.tokens));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int here = cached - h * kKeys;
                  unsigned long long word = ~0ull;
                  if (here < kKeys) word = here > 0 ? drafted << here | ((1ull << here) - 1) : here > -64 ? drafted >> -here : 0ull;
                  if (hidden) {
                    for (int i = 0; i < min(here, kKeys); ++i)
                      if ((unsigned)page_of(p, seg, (tile + h) * kKeys + i) >= (unsigned)a.pages) word &= ~(1ull << i);
                  }
                  sees[2 * h] = (uint32_t)word;
                  sees[2 * h + 1] = (uint32_t)(word >> 32);
                }
              }
              auto hide = [&](uint32_t* s, int c) {
                if constexpr (kHides) {
                  const uint32_t word = c == 0 ? sees[0] : c == 1 ? sees[1] : c == 2 ? sees[2] : sees[3];
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (!(word >> i & 1)) s[i] = __float_as_uint(-INFINITY);
                }
              };
              uint32_t v0[32], v1[32];
              float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
              auto largest = [&](uint32_t* s, int c) {
                hide(s, c);
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                  m0 = fmaxf(m0, fmaxf(as_float(s[i]), as_float(s[i + 1])));
                  m1 = fmaxf(m1, fmaxf(as_float(s[i + 2]), as_float(s[i + 3])));
                  m2 = fmaxf(m2, fmaxf(as_float(s[i + 4]), as_float(s[i + 5])));
                  m3 = fmaxf(m3, fmaxf(as_float(s[i + 6]), as_float(s[i + 7])));
                }
              };
              tmem_load<32>(my_scores, v0);
#pragma unroll 1
              for (int c = 0; c < chunks; c += 2) {
                tmem_loaded<32>(v0);
                tmem_load<32>(my_scores + 32 * (c + 1), v1);
                largest(v0, c);
                tmem_loaded<32>(v1);
                tmem_load<32>(my_scores + 32 * (c + 2 < chunks ? c + 2 : 0), v0);        // (the last one: the first again)
                largest(v1, c + 1);
              }
              const float m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * sl;
              if (__any_sync(0xffffffffu, m > top + kGrowth || (top == -INFINITY && m > top))) {
                const float now = fmaxf(top, m);
                const float keep = exp2_approx(top - (now == -INFINITY ? 0.f : now));
                top = now;
                total *= keep;
                rounds = __any_sync(0xffffffffu, fabsf(top) >= 4194304.f);
                if (any) {
                  // (the product before these scores is done: the tensor cores work in the order of issue)
#pragma unroll 1
                  for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
                    tmem_load<16>(my_sums + c, o);
                    tmem_loaded<16>(o);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(as_float(o[i]) * keep);
                    tmem_store16(my_sums + c, o);
                  }
                }
              }
              if (!kHides && rounds) {
                tmem_loaded<32>(v0);
                return false;
              }
              const float before = kHides && rounds ? sl : 1.f, within = kHides && rounds ? 1.f : sl;      // scores are multiplied by, rounded, and by
              const float base_log2 = top == -INFINITY ? 0.f : top;
              float t0 = 0.f, t1 = 0.f, t2 = 0.f, t3 = 0.f;
              auto exponentials = [&](uint32_t* s, int c) {
                hide(s, c);
                auto weight = [&](uint32_t score) { return exp2_approx(fmaf(kHides ? as_float(score) * before : as_float(score), within, -base_log2)); };
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const float e0 = weight(s[i]), e1 = weight(s[i + 1]), e2 = weight(s[i + 2]), e3 = weight(s[i + 3]);
                  t0 += e0;
                  t1 += e1;
                  t2 += e2;
                  t3 += e3;
                  w[i / 2] = Half16<T>::pack(e0, e1);
                  w[i / 2 + 1] = Half16<T>::pack(e2, e3);
                }
                tmem_store16(my_scores + 16 * c, w);                 // over scores that have been read
              };
#pragma unroll 1
              for (int c = 0; c < chunks; c += 2) {
                tmem_loaded<32>(v0);
                tmem_load<32>(my_scores + 32 * (c + 1), v1);
                exponentials(v0, c);
                tmem_loaded<32>(v1);
                if (c + 2 < chunks) tmem_load<32>(my_scores + 32 * (c + 2), v0);
                exponentials(v1, c + 1);
              }
              total += (t0 + t1) + (t2 + t3);
              return true;
            };
            if (cached < chunks * 32 || hidden || rounds || !weigh(std::false_type())) weigh(std::true_type());
            tc_wait_st();
          }
          any = true;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(weights + 8 * group);
          ++job;
        }
        if (kPair && !group_lives) continue;

        // ---- the end of a segment
        if (any) {
          mbar_wait_bounded<20>(product + 8 * group, ended++ & 1, p.status, dead);
          tc_fence_after();
        }
        const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
        float* slot = nullptr;
        constexpr int kGroups = kPair ? 2 : 1;                       // that leave a partial
        const int which = kPair ? group : 0;
        auto slot_of = [&](int c, bool first) { return p.partials + ((size_t)(c * kGroups + which) * 2 + (first ? 1 : 0)) * C::kSlotFloats; };
        if (!whole) slot = slot_of(cta, seg.t0 == 0);
        float mine = 1.f, theirs = 0.f;
        if (!kPair) {
          // the second group hands its maxima, totals and sums to the first
          if (group == 1 && row_in >= 0) {
            stats[row_in] = top;
            stats[kRowTile + row_in] = total;
          }
          named_bar_sync(1, 256);
          if (group == 0) {
            const float other = stats[row_in], both = fmaxf(top, other), base_log2 = both == -INFINITY ? 0.f : both;
            mine = exp2_approx(top - base_log2);
            theirs = exp2_approx(other - base_log2);
            total = total * mine + stats[kRowTile + row_in] * theirs;
            top = both;
          }
        }
        bool odd = odd_ring[segment % kOddRing] != 0;                // (both groups' products are done)
        const bool none = mask == 0 || total == 0.f;                 // padding, and rows that see nothing, are zero
        const float f = 1.f / total;
        T* out = static_cast<T*>(a.out) + seg.b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2];
        // infinite and NaN values of drafted tokens, for the rows that see them
        auto add_odd = [&](float (&v)[32], int c) {
          for (int j = 0; j < a.tokens; ++j) {
            if (!(mask >> j & 1)) continue;
            const uint16_t* from = static_cast<const uint16_t*>(a.v) + seg.b * a.v_stride[0] + j * a.v_stride[1] + g * a.v_stride[2] + c;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((from[i] & Half16<T>::kExponent) == Half16<T>::kExponent) v[i] += Half16<T>::value(from[i]);
          }
        };
        auto put = [&](float (&v)[32], int c, float by, bool zero, bool add) {
          if (!row_lives) return;
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] *= by;
          if (add) add_odd(v, c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = zero ? 0u : Half16<T>::pack(v[8 * i + 2 * e], v[8 * i + 2 * e + 1]);
            *reinterpret_cast<uint4*>(out + c + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        };
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          if (any && warp_lives) {
            tmem_load<32>(my_sums + c0, o);
            tmem_loaded<32>(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (!kPair) {
            if (group == 1 && row_in >= 0) {
#pragma unroll
              for (int i = 0; i < 8; ++i) exchange[i * kRowTile + row_in] = make_float4(as_float(o[4 * i]), as_float(o[4 * i + 1]), as_float(o[4 * i + 2]), as_float(o[4 * i + 3]));
            }
            named_bar_sync(1, 256);
          }
          if ((kPair || group == 0) && warp_lives) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = as_float(o[i]) * mine;
            if (!kPair) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 x = exchange[i * kRowTile + row_in];
                v[4 * i] = fmaf(x.x, theirs, v[4 * i]);
                v[4 * i + 1] = fmaf(x.y, theirs, v[4 * i + 1]);
                v[4 * i + 2] = fmaf(x.z, theirs, v[4 * i + 2]);
                v[4 * i + 3] = fmaf(x.w, theirs, v[4 * i + 3]);
              }
            }
            if (whole) {
              put(v, c0, f, none, odd);
            } else {
              float4* to = reinterpret_cast<float4*>(slot) + c0 / 4 * kRowTile + row_in;
#pragma unroll
              for (int i = 0; i < 8; ++i) __stcg(to + i * kRowTile, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
            }
          }
          if (!kPair) named_bar_sync(1, 256);
        }
        if (whole || (!kPair && group == 1)) continue;
        slot[kRowTile * D + row_in] = top;
        slot[kRowTile * (D + 1) + row_in] = total;
        if (row_in == 0) reinterpret_cast<int*>(slot)[kRowTile * (D + 2)] = odd;
        const int first_cta = seg.t0 == 0 ? cta : cta_of(units, ctas, seg.unit + p.overhead);
        const int last_cta = cta_of(units, ctas, seg.unit + p.overhead + seg.tiles - 1);
        const Joining join(first_cta, last_cta, cta, join_step(last_cta - first_cta + 1));
        // whether this CTA is the last of those that a counter waits for; what the others wrote is visible then
        auto last_at = [&](unsigned int* counter, int others) {
          __threadfence();
          named_bar_sync(4 + which, 128);
          if (row_in == 0) {
            const bool is_last = atomicAdd(counter, 1u) == (unsigned)others;
            if (is_last) *counter = 0;                               // for the next launch
            misc[2 + which] = is_last;
          }
          named_bar_sync(4 + which, 128);
          const bool is_last = misc[2 + which] != 0;
          __threadfence();
          return is_last;
        };
        // Up to 64 rows, two threads share a row when partials are joined.
        const bool shared = q_sets == 2;
        const int join_row = shared ? row_in & 63 : row_in, c_begin = shared ? row_in / 64 * (D / 2) : 0, c_end = shared ? c_begin + D / 2 : D;
        // Joins `count` partials, `step` CTAs apart: into the output, or into the first one's slot.
        auto add_up = [&](int c0, int count, int step, bool ends) {
          const int last = c0 + (count - 1) * step;
          auto from = [&](int k) {
            const int c = min(c0 + k * step, last);
            return slot_of(c, c == first_cta);
          };
          float m = -INFINITY, sum = 0.f;
          bool odd = false;
          for (int k = 0; k < count; k += 4) {
            float cm[4], ct[4], most = m;
            int any_odd = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float* at = from(k + e);
              cm[e] = __ldcg(at + kRowTile * D + join_row);
              ct[e] = __ldcg(at + kRowTile * (D + 1) + join_row);
              any_odd |= __ldcg(reinterpret_cast<const int*>(at) + kRowTile * (D + 2));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k + e < count) most = fmaxf(most, cm[e]);
            const float base_log2 = most == -INFINITY ? 0.f : most;
            sum *= exp2_approx(m - base_log2);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k + e < count) sum += ct[e] * exp2_approx(cm[e] - base_log2);
            m = most;
            odd = odd || any_odd != 0;
          }
          const float base_log2 = m == -INFINITY ? 0.f : m;
          float* to = slot_of(c0, c0 == first_cta);
          if (row_tile * kRowTile + join_row < p.rows) {
#pragma unroll 1
            for (int c = c_begin; c < c_end; c += 32) {
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
              // (two contributors at a time: what this takes is the latency of its loads)
#pragma unroll 1
              for (int k = 0; k < count; k += 2) {
                float by[2];
                float4 x[2][8];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float4* at = reinterpret_cast<const float4*>(from(k + e)) + c / 4 * kRowTile + join_row;
                  by[e] = __ldcg(from(k + e) + kRowTile * D + join_row);
#pragma unroll
                  for (int i = 0; i < 8; ++i) x[e][i] = __ldcg(at + i * kRowTile);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  if (k + e >= count) continue;
                  const float f = exp2_approx(by[e] - base_log2);
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    v[4 * i] = fmaf(x[e][i].x, f, v[4 * i]);
                    v[4 * i + 1] = fmaf(x[e][i].y, f, v[4 * i + 1]);
                    v[4 * i + 2] = fmaf(x[e][i].z, f, v[4 * i + 2]);
                    v[4 * i + 3] = fmaf(x[e][i].w, f, v[4 * i + 3]);
                  }
                }
              }
              if (ends) {
                put(v, c, 1.f / sum, mask == 0 || sum == 0.f, odd);
              } else {
                float4* at = reinterpret_cast<float4*>(to) + c / 4 * kRowTile + join_row;
#pragma unroll
                for (int i = 0; i < 8; ++i) __stcg(at + i * kRowTile, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
              }
            }
          }
          if (ends) return;
          named_bar_sync(4 + which, 128);                            // all have read the first one's maxima
          if (c_begin == 0) {
            __stcg(to + kRowTile * D + join_row, m);
            __stcg(to + kRowTile * (D + 1) + join_row, sum);
            if (row_in == 0) __stcg(reinterpret_cast<int*>(to) + kRowTile * (D + 2), odd ? 1 : 0);
          }
        };
        if (shared) {
          // the row that this thread joins, in place of its own
          row_lives = join_row < p.rows;
          const int join_t = row_lives ? join_row / p.group : 0;
          mask = row_lives ? mask_of(p, seg.b, join_t) : 0;
          out = static_cast<T*>(a.out) + seg.b * a.out_stride[0] + join_t * a.out_stride[1] + (g * p.group + (row_lives ? join_row - join_t * p.group : 0)) * a.out_stride[2];
        }
        // (one loop, so that its code is there once: what runs for the first time takes longer to fetch than to run)
        const bool grouped = join.step < join.count;
        bool ends = !grouped;
#pragma unroll 1
        while (last_at(ends && grouped ? join.item_counter(p, which) : join.group_counter(p, which), (ends && grouped ? join.groups() : join.size) - 1)) {
          add_up(ends ? first_cta : join.group, ends && grouped ? join.groups() : join.size, ends && grouped ? join.step : 1, ends);
          if (ends) break;
          ends = true;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && misc[1] && p.status) atomicExch(p.status, FP6M_ERR_BAD_ARG);
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <class T, class C, class Scales>
cudaError_t launch_tc5(const TreeParams& p, const Scales& scales, int ctas, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
  cudaError_t e = allow_shared_memory<tree_attention_tc5_kernel<T, C, Scales>>(C::kSmemBytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(tree_attention_tc5_kernel<T, C, Scales>, dim3(ctas), dim3(kTreeThreads), C::kSmemBytes, stream, p, scales, kmap, vmap);
}
template <class T, class Scales>
cudaError_t launch_typed(const TreeParams& p, const Scales& scales, int ctas, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
  constexpr bool kFp8 = !std::is_same<Scales, NoScales>::value;
  const bool pair = p.row_tiles > 1;
  if (p.a.head_dim == 64) return pair ? launch_tc5<T, TreeCfg<64, true, kFp8>>(p, scales, ctas, kmap, vmap, stream) : launch_tc5<T, TreeCfg<64, false, kFp8>>(p, scales, ctas, kmap, vmap, stream);
  return pair ? launch_tc5<T, TreeCfg<128, true, kFp8>>(p, scales, ctas, kmap, vmap, stream) : launch_tc5<T, TreeCfg<128, false, kFp8>>(p, scales, ctas, kmap, vmap, stream);
}

}  // namespace

// (a CTA leaves at most two partials for each of two row tiles)
size_t tree_tc5_partial_bytes(int sms) { return (size_t)(sms > 0 && sms < kMostTreeCtas ? sms : kMostTreeCtas) * 4 * TreeCfg<128, true>::kSlotFloats * sizeof(float); }

cudaError_t launch_tree_tc5(TreeParams p, const fp6m_cache_scales* scales, int sms, cudaStream_t stream) {
  p.row_tiles = (p.rows + kRowTile - 1) / kRowTile;
  p.parts = (p.row_tiles + 1) / 2;
  p.overhead = 4;
  const int ctas = sms < kMostTreeCtas ? sms : kMostTreeCtas;
  // the tokens that lie next to one another in a page and start at a multiple of their number in a tile: swizzled rows need eight
  const fp6m_tree_attention_args& a = p.a;
  p.run = kKeys;
  while (a.page_size % p.run) p.run /= 2;
  CUtensorMap kmap = {}, vmap = {};
  auto encode = [&](const void* cache, const long long (&strides)[3], CUtensorMap* map) {
    return scales ? encode_plain_cache_map(cache, a.head_dim, a.kv_heads, a.page_size, a.pages, strides, p.run, map)
                  : encode_cache_map(cache, 2, a.head_dim, a.kv_heads, a.page_size, a.pages, strides, p.run, map);
  };
  if (p.run < 8 || a.max_pages == 0 || encode(a.k_cache, a.k_cache_stride, &kmap) != cudaSuccess || encode(a.v_cache, a.v_cache_stride, &vmap) != cudaSuccess) p.run = 0;
  const bool is_half = a.type == FP6M_TYPE_F16;
  if (scales) return is_half ? launch_typed<half>(p, *scales, ctas, kmap, vmap, stream) : launch_typed<__nv_bfloat16>(p, *scales, ctas, kmap, vmap, stream);
  return is_half ? launch_typed<half>(p, NoScales(), ctas, kmap, vmap, stream) : launch_typed<__nv_bfloat16>(p, NoScales(), ctas, kmap, vmap, stream);
}

}  // namespace fp6m
