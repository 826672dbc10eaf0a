// C = A B^T of E4M3 matrices with scales for blocks of 128, more than 64 rows of A: see mul_fp8.cu for the product itself.
//
// Here the rows of A are the lanes of the accumulators: a thread sums columns of one row of C, so a block of K has one scale per
// thread - sa of its row times sb of its columns - and not one per value.  More than 128 rows: two CTAs share a tile of 256 rows
// and 256 columns (cta_group::2).  Each brings 128 rows of A and half of the columns of B, 32 KB per block of K for 512 cycles of
// the tensor cores; one CTA alone would have to bring 48 KB, more than the 64 bytes a cycle that reach a multiprocessor.
// Up to 128 rows: one CTA, 128 columns.
//
// Every pair of CTAs (or CTA) computes whole tiles, in the order of the tiles, as long as all have one.  What is left is cut along K
// into equal ranges if that shortens the end by more than the exchange of their sums takes: all leave theirs in the scratch, and the
// CTA that does so last adds them in the order of the ranges (an arrival counter; nobody waits).
//
// 4096 rows, 8192 x 28672 (K x N), public calls one behind the other: 942 us, 2040 TFLOP/s, 1.22 times what a library product in bf16 reaches.  A block takes a pair 875 cycles, of which the tensor cores
// work 512: between them lies the sums' way (256 read-backs, 256 multiply-adds and the barriers per thread and block), which two accumulator tiles - all that tensor
// memory holds of 256 columns - do not hide in full, and the clock falls to about 1.6 GHz under the power limit.  131 rows, 11008 x 4096: 25.4 us where the bytes
// take 7: two row tiles of 32 KB a block each (37 blocks of 540 cycles), set-up and first data (7500 cycles), exchange (10000).
#include "../../include/fp6m.h"
#include "host_common.h"
#include "mul_fp8.cuh"

namespace fp6m {

namespace {

constexpr int kMaxTeams = kMaxFp8Ctas;

struct RowsParams {
  void* C;
  const float *sa, *sb;
  int M, N, kb;
  int row_tiles, tiles;                  // tiles in the order of their columns, row tiles next to one another
  int whole;                             // whole tiles of every team
  int extra;                             // the first teams that take one more, if the tiles that are left are not cut
  int sharers;                           // teams that share the tiles that are left, cut along K (0: see extra)
  int weights_early;
  unsigned int* arrived;                 // [CTA] sums that were left for the tile that starts in that CTA's range
  float4* partials;                      // [CTA][2][warp][4 columns][lane]: sums of a tile that starts before, in, the CTA's range
  int* status;
};

// kGroup CTAs (1 or 2) form a team with a tile of 128 * kGroup rows and columns.
template <int GROUP_>
struct RowsCfg {
  static constexpr int kGroup = GROUP_;
  static constexpr int kColumns = 128 * kGroup;              // of a tile
  static constexpr int kStageBytes = 2 * kStripBytes;        // 128 rows of A, 128 columns of B
  static constexpr int kStages = 6;
  static constexpr int kTiles = 512 / kColumns;              // accumulator tiles in tensor memory
  static constexpr int kMine = kColumns / 2;                 // columns of a thread
  static constexpr int kWarps = 8;
  static constexpr int kThreads = 32 * (4 + kWarps);
  static constexpr int kAhead = 8;                           // blocks of K whose scales are brought together
  static constexpr int kScalePitch = 132;                    // floats from one block's row scales to the next: no bank conflicts
  static constexpr int kScaleFloats = kAhead * (kScalePitch + 2);
  static constexpr int kNumBars = 2 * kStages + 2 * kTiles + 4;
  static constexpr int kOutRow = 32 * 2 + 16;                // bytes of a row of 32 finished values in shared memory, with a gap
  static constexpr int kSmemBytes = kStages * kStageBytes + kWarps * 32 * kOutRow + 2 * kScaleFloats * 4 + kNumBars * 8 + 16 + 1024;
  static constexpr int kSlotFloat4 = kWarps * kMine / 4 * 32;
};

// A team's work: segments of one tile and a range of blocks of K each.
struct Segments {
  int team, teams, index = 0;
  long long u, end;                      // of the tiles that are shared
  __device__ __forceinline__ Segments(const RowsParams& p, int team_, int teams_) : team(team_), teams(teams_) {
    u = start_of(p, team);
    end = start_of(p, team + 1);
  }
  // The start of a team's range among the blocks of the shared tiles.
  static __device__ __forceinline__ long long start_of(const RowsParams& p, int team, int teams) {
    return p.sharers ? (long long)(p.tiles - p.whole * teams) * p.kb * min(team, p.sharers) / p.sharers : 0;
  }
  __device__ __forceinline__ long long start_of(const RowsParams& p, int t) const { return start_of(p, t, teams); }
  __device__ __forceinline__ bool next(const RowsParams& p, int& tile, int& k0, int& k1) {
    if (index < p.whole + (team < p.extra)) {
      tile = team + teams * index++;
      k0 = 0;
      k1 = p.kb;
      return true;
    }
    if (u >= end) return false;
    const int in = (int)(u / p.kb);
    tile = p.whole * teams + in;
    k0 = (int)(u - (long long)in * p.kb);
    const long long stop = min((long long)(in + 1) * p.kb, end);
    k1 = (int)(stop - (long long)in * p.kb);
    u = stop;
    return true;
  }
};

__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {       // the same place in the shared memory of the team's first CTA
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// A copy into this CTA that is counted by a barrier of the team's first CTA.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int row, uint32_t leader_bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(leader_bar) : "memory");
}
template <int kGroup>
__device__ __forceinline__ void mma_tile(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kGroup == 1)
      asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
                   ::"r"(d_tmem), "l"(a_desc + 2 * i), "l"(b_desc + 2 * i), "r"(idesc), "r"(i) : "memory");
    else
      asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
                   ::"r"(d_tmem), "l"(a_desc + 2 * i), "l"(b_desc + 2 * i), "r"(idesc), "r"(i) : "memory");
  }
}
// Arrives at the barrier (in both CTAs of a pair, at the same place) when the MMAs issued so far are done.
template <int kGroup>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (kGroup == 1) {
    tc_commit(bar);
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  }
}
template <class T> struct Two;
template <> struct Two<half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) { half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
};
template <> struct Two<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) { __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
};

template <class T, class C>
__global__ void __launch_bounds__(C::kThreads, 1)
mul_fp8_rows_kernel(const __grid_constant__ RowsParams p, const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap) {
  constexpr int S = C::kStages, D = C::kTiles, G = C::kGroup;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* out_stage = smem + S * C::kStageBytes;                                   // [warp][32 rows][kOutRow]
  float* scales = reinterpret_cast<float*>(out_stage + C::kWarps * 32 * C::kOutRow);    // [2]: [block][row], then [block][128 columns]
  uint64_t* bars = reinterpret_cast<uint64_t*>(scales + 2 * C::kScaleFloats);
  volatile uint32_t* misc = reinterpret_cast<uint32_t*>(bars + C::kNumBars);        // [0] TMEM base, [1] this CTA arrived last
  const uint32_t full = smem_u32(bars), empty = full + 8 * S, done = empty + 8 * S, taken = done + 8 * D, scaled = taken + 8 * D, used = scaled + 16;

  const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31;
  const int rank = G == 1 ? 0 : blockIdx.x & 1;              // in the team (clusters are neighbouring CTAs)
  const int teams = gridDim.x / G, team = (int)blockIdx.x / G;
  launch_dependents();

  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full + 8 * s, 1);                            // the expect_tx arrival of the first CTA's producer
      mbar_init(empty + 8 * s, 1);                           // tcgen05.commit: the block's MMAs have read the stage
    }
    for (int d = 0; d < D; ++d) {
      mbar_init(done + 8 * d, 1);                            // tcgen05.commit: the tile holds the block's products
      mbar_init(taken + 8 * d, G * C::kWarps);               // the warps of the team have read it back (in the first CTA)
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(scaled + 8 * i, 1);
      mbar_init(used + 8 * i, C::kWarps);
    }
    mbar_fence_init();
  }
  if (warp == 3) {
    if constexpr (G == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(const_cast<uint32_t*>(misc))) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(const_cast<uint32_t*>(misc))) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cluster_sync();                      // the barriers of both CTAs exist
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, misc[0], 0);
  bool dead = false;
  // The launch gives 168 registers a thread (384 threads); the eight warps that hold sums take 216, the first four keep 72:
  // 256 * 216 + 128 * 72 = 384 * 168.
  Segments segments(p, team, teams);
  int tile, k0, k1;

  if (warp == 0) {
    // ================================================================== producer: this CTA's rows of A and columns of B
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const uint32_t bar0 = G == 1 ? full : in_leader(full);
    auto load = [&](const CUtensorMap* map, uint32_t dst, int x, int row, uint32_t bar) {
      if constexpr (G == 1) tma_load_bytes(dst, map, x, row, bar);
      else tma_load_pair(dst, map, x, row, bar);
    };
    // the first round of stages is free; its weights come into L2 while the kernel in front finishes, or are copied if they may be
    Segments ahead = segments;
    int n = 0;
    while (n < S && ahead.next(p, tile, k0, k1))
      for (int k = k0; k < k1 && n < S; ++k, ++n)
        if (elect_one()) {
          const int column = (tile / p.row_tiles) * C::kColumns + rank * 128;
          if (!p.weights_early) {
            tma_prefetch_bytes(&bmap, k * kBlock, column);
          } else {
            if (rank == 0) mbar_arrive_expect_tx(full + 8 * n, G * C::kStageBytes);
            load(&bmap, smem_u32(smem) + n * C::kStageBytes + kStripBytes, k * kBlock, column, bar0 + 8 * n);
          }
        }
    __syncwarp();
    grid_dependency_wait();
    int stage = 0;
    uint32_t phase = 0;
    bool first = true;                                       // the first round
    while (segments.next(p, tile, k0, k1)) {
      const int row = tile % p.row_tiles * (128 * G) + rank * 128, column = (tile / p.row_tiles) * C::kColumns + rank * 128;
      for (int k = k0; k < k1; ++k) {
        if (!first) mbar_wait_bounded<50>(empty + 8 * stage, phase ^ 1, p.status, dead);
        if (elect_one()) {
          const uint32_t dst = smem_u32(smem) + stage * C::kStageBytes;
          if (!first || !p.weights_early) {
            if (rank == 0) mbar_arrive_expect_tx(full + 8 * stage, G * C::kStageBytes);
            load(&bmap, dst + kStripBytes, k * kBlock, column, bar0 + 8 * stage);
          }
          load(&amap, dst, k * kBlock, row, bar0 + 8 * stage);
        }
        __syncwarp();
        if (++stage == S) { stage = 0; phase ^= 1; first = false; }
      }
    }
    // no arrival of the last MMAs is on its way to this CTA when it ends
    for (int n = 0; n < S; ++n) {
      if (!first) mbar_wait_bounded<50>(empty + 8 * stage, phase ^ 1, p.status, dead);
      else if (n < stage) mbar_wait_bounded<50>(empty + 8 * n, 0, p.status, dead);
      if (!first && ++stage == S) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    // ================================================================== MMA issuer, in the first CTA of the team
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    grid_dependency_wait();                                  // the bounded waits start when the kernel in front has finished
    if (rank == 0) {
      const uint64_t desc0 = wide_act_desc(smem_u32(smem));
      // D fp32, A and B E4M3, K-major; N = columns, M = 128 rows per CTA
      constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(C::kColumns >> 3) << 17) | ((uint32_t)(128 * G >> 4) << 24);
      int stage = 0, buffer = 0;
      uint32_t phase = 0, tphase = 0;
      while (segments.next(p, tile, k0, k1))
        for (int k = k0; k < k1; ++k) {
          mbar_wait_bounded<20>(taken + 8 * buffer, tphase ^ 1, p.status, dead);
          mbar_wait_bounded<20>(full + 8 * stage, phase, p.status, dead);
          tc_fence_after();
          // the descriptor's low 14 bits hold the address / 16: adding an offset never carries out of them
          const uint64_t a_desc = desc0 + (uint64_t)(stage * (C::kStageBytes >> 4));
          if (elect_one()) {
            mma_tile<G>(tmem + buffer * C::kColumns, a_desc, a_desc + (kStripBytes >> 4), idesc);
            commit<G>(empty + 8 * stage);
            commit<G>(done + 8 * buffer);
          }
          __syncwarp();
          if (++stage == S) { stage = 0; phase ^= 1; }
          if (++buffer == D) { buffer = 0; tphase ^= 1; }
        }
    }
  } else if (warp == 2) {
    // ================================================================== scales, of eight blocks of K at a time
    // (Loaded by the warps that sum, a row and block a lane, they cost those warps 280 cycles a block.)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    grid_dependency_wait();
    constexpr int A = C::kAhead;
    const int block = lane % A, row_of_lane = lane / A, step = 32 / A;
    int turn = 0;
    uint32_t phase = 0;
    while (segments.next(p, tile, k0, k1)) {
      const int row0 = tile % p.row_tiles * (128 * G) + rank * 128;
      const int strip = min((tile / p.row_tiles) * G + (lane / A) % G, (p.N - 1) / kBlock);
      for (int k = k0; k < k1; k += A) {
        const bool live = k + block < k1;
        float row_scale[128 / step];
#pragma unroll
        for (int i = 0; i < 128 / step; ++i) {
          const int row = row0 + row_of_lane + step * i;
          row_scale[i] = live && row < p.M ? p.sa[(size_t)row * p.kb + k + block] : 0.f;
        }
        const float strip_scale = live ? p.sb[(size_t)strip * p.kb + k + block] : 0.f;
        float* to = scales + turn * C::kScaleFloats;
        mbar_wait_bounded<100>(used + 8 * turn, phase ^ 1, p.status, dead);
#pragma unroll
        for (int i = 0; i < 128 / step; ++i) sts_f32(smem_u32(to + block * C::kScalePitch + row_of_lane + step * i), row_scale[i]);
        if (lane < A * G) sts_f32(smem_u32(to + A * C::kScalePitch + block * G + lane / A), strip_scale);
        __syncwarp();
        if (lane == 0) mbar_arrive(scaled + 8 * turn);
        turn ^= 1;
        if (turn == 0) phase ^= 1;
      }
    }
  } else if (warp == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    grid_dependency_wait();
  } else {
    // ================================================================== sums: thread = row of the tile, kMine columns
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    constexpr int E = C::kMine;
    const int quarter = warp & 3, half_index = (warp - 4) >> 2;
    const int row_in = quarter * 32 + lane, column_in = half_index * E;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + column_in;
    const uint32_t taken0 = G == 1 ? taken : in_leader(taken);
    grid_dependency_wait();
    float sum[E];
    int buffer = 0, turn = 0;
    uint32_t tphase = 0, sphase = 0;
    // A warp turns 32 rows x 32 columns at a time round in shared memory: four lanes store 64 bytes of a row.
    uint8_t* mine = out_stage + (warp - 4) * 32 * C::kOutRow;
    auto put = [&](const float* v, int row0, int column0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = Two<T>::pack(v[i * 8 + 2 * e], v[i * 8 + 2 * e + 1]);
        *reinterpret_cast<uint4*>(mine + lane * C::kOutRow + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncwarp();
      const int column = column0 + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2);
        if (row0 + r < p.M && column < p.N)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.C) + (size_t)(row0 + r) * p.N + column) = *reinterpret_cast<const uint4*>(mine + r * C::kOutRow + (lane & 3) * 16);
      }
      __syncwarp();
    };
    while (segments.next(p, tile, k0, k1)) {
#pragma unroll
      for (int i = 0; i < E; ++i) sum[i] = 0.f;
#pragma unroll 1
      for (int k = k0; k < k1; k += C::kAhead) {
        mbar_wait_bounded<20>(scaled + 8 * turn, sphase, p.status, dead);
        const uint32_t row_scale = smem_u32(scales + turn * C::kScaleFloats + row_in);
        const uint32_t strip_scale = smem_u32(scales + turn * C::kScaleFloats + C::kAhead * C::kScalePitch + (G == 1 ? 0 : half_index));
        const int blocks = min(C::kAhead, k1 - k);
#pragma unroll 1
        for (int j = 0; j < blocks; ++j) {
          const float scale = lds_f32(row_scale + j * C::kScalePitch * 4) * lds_f32(strip_scale + j * G * 4);
          mbar_wait_bounded<20>(done + 8 * buffer, tphase, p.status, dead);
          tc_fence_after();
          const uint32_t from = lane_base + buffer * C::kColumns;
          // 32 columns are on their way while 32 are added; the tile is given back before the last ones are
          uint32_t v[2][32];
          tmem_load<32>(from, v[0]);
#pragma unroll
          for (int c = 0; c < E / 32; ++c) {
            tmem_loaded<32>(v[c & 1]);
            if (c + 1 < E / 32) {
              tmem_load<32>(from + 32 * (c + 1), v[(c + 1) & 1]);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if constexpr (G == 1) mbar_arrive(taken0 + 8 * buffer);
                else arrive_at(taken0 + 8 * buffer);
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c * 32 + i] = fmaf(__uint_as_float(v[c & 1][i]), scale, sum[c * 32 + i]);
          }
          if (++buffer == D) { buffer = 0; tphase ^= 1; }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(used + 8 * turn);
        turn ^= 1;
        if (turn == 0) sphase ^= 1;
      }
      // ---- the end of a segment
      const int row0 = tile % p.row_tiles * (128 * G) + rank * 128 + quarter * 32, column0 = (tile / p.row_tiles) * C::kColumns + column_in;
      if (k0 == 0 && k1 == p.kb) {
#pragma unroll
        for (int c = 0; c < E / 32; ++c) put(sum + c * 32, row0, column0 + c * 32);
        continue;
      }
      // Part of a tile.  Only a team's first segment of the shared tiles can start inside a tile, only its last one can end inside.
      constexpr int kPart = E / 4 * 32;
      auto slot_of = [&](int t, int which) { return p.partials + ((size_t)(t * G + rank) * 2 + which) * C::kSlotFloat4 + (warp - 4) * kPart + lane; };
      float4* slot = slot_of(team, k0 == 0 ? 1 : 0);
#pragma unroll
      for (int i = 0; i < E / 4; ++i) __stcg(slot + i * 32, make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]));
      const long long begin = (long long)(tile - p.whole * teams) * p.kb, end = begin + p.kb;
      int first = team, last = team;
      while (segments.start_of(p, first) > begin) --first;
      while (last + 1 < p.sharers && segments.start_of(p, last + 1) < end) ++last;
      __threadfence();
      named_bar_sync(1, C::kWarps * 32);
      if (tid == 128) {
        const bool is_last = atomicAdd(p.arrived + first * G + rank, 1u) == (unsigned)(last - first);
        if (is_last) p.arrived[first * G + rank] = 0;        // for the next launch
        misc[1] = is_last;
      }
      named_bar_sync(1, C::kWarps * 32);
      if (misc[1]) {
        __threadfence();
#pragma unroll 1
        for (int c = 0; c < E / 32; ++c) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
          // (four contributors on their way at a time: with one the loads' latency made this 20,000 cycles for six of them)
#pragma unroll 1
          for (int t = first; t <= last; t += 4) {
            float4 w[4][8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4* from = slot_of(min(t + e, last), t + e == first ? 1 : 0) + c * 8 * 32;
#pragma unroll
              for (int i = 0; i < 8; ++i) w[e][i] = t + e <= last ? __ldcg(from + i * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                v[4 * i] += w[e][i].x;
                v[4 * i + 1] += w[e][i].y;
                v[4 * i + 2] += w[e][i].z;
                v[4 * i + 3] += w[e][i].w;
              }
          }
          put(v, row0, column0 + c * 32);
        }
      }
      named_bar_sync(1, C::kWarps * 32);                     // all have read the answer
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cluster_sync();                      // nothing of the other CTA's arrives here any more
  tc_fence_after();
  if (warp == 3) {
    if constexpr (G == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

struct RowsPlan {
  int group, row_tiles, tiles, teams, whole, extra, sharers;
  double cost;
};
// One CTA or two per team, and whether the tiles that are left after the whole ones are cut along K: what takes the least time, in blocks of a single
// CTA (540 cycles; a pair of CTAs takes 1.6 times that for four times the work).  An exchange of sums, from their store to the last result, took
// as long as 26 blocks where a CTA has 128 x 128 of them, and as 56 with 128 x 256.  us with teams of one / two (shared or not as this rule
// has it): 131 x 11008 x 4096 24 / 31, 256 x 4096 x 4096 13.6 / 26, 400 x 8192 x 8192 46 / 34, 512 x 4096 x 11008 37 / 42, 777 x 4096 x 11008
// 55 / 54, 1024 x 4096 x 4096 24 / 20, 2048 x 8192 x 8192 150 / 127 (rows x K x columns).
RowsPlan plan_teams(int group, int M, int N, int K, int sms) {
  RowsPlan plan;
  plan.group = group;
  const int edge = 128 * group, kb = (K + kBlock - 1) / kBlock;
  const double block = group == 1 ? 1.0 : 1.6, exchange = group == 1 ? 26 : 56;
  plan.row_tiles = (M + edge - 1) / edge;
  plan.tiles = plan.row_tiles * ((N + edge - 1) / edge);
  plan.teams = (sms > 0 && sms < kMaxFp8Ctas ? sms : kMaxFp8Ctas) / group;
  if (plan.teams < 1) plan.teams = 1;
  plan.whole = plan.tiles / plan.teams;
  const int left = plan.tiles - plan.whole * plan.teams;
  plan.extra = left;
  plan.sharers = 0;
  plan.cost = (plan.whole + (left > 0)) * (double)kb * block;
  if (left > 0) {
    const long long blocks = (long long)left * kb;
    const int sharers = (int)(blocks / 4 < plan.teams ? (blocks + 3) / 4 : plan.teams);      // at least four blocks each
    const double shared = ((double)plan.whole * kb + (double)((blocks + sharers - 1) / sharers)) * block + exchange;
    if (shared < plan.cost) {
      plan.cost = shared;
      plan.extra = 0;
      plan.sharers = sharers;
    }
  }
  if (plan.whole == 0) plan.teams = plan.sharers ? plan.sharers : left;
  return plan;
}
RowsPlan plan_rows(int M, int N, int K, int sms) {
  const RowsPlan one = plan_teams(1, M, N, K, sms);
  if (M <= 128) return one;
  const RowsPlan two = plan_teams(2, M, N, K, sms);
  return two.cost < one.cost ? two : one;
}
size_t rows_bytes(const RowsPlan& plan) {
  return plan.sharers ? kRowsScratch + (size_t)plan.teams * plan.group * 2 * (plan.group * 64) * 256 * sizeof(float) : kRowsScratch;
}

template <class T, int kGroup>
cudaError_t launch_rows(const RowsParams& p, int teams, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  using C = RowsCfg<kGroup>;
  static_assert(C::kSlotFloat4 * 4 == kGroup * 64 * 256, "slot");
  cudaError_t e = allow_shared_memory<mul_fp8_rows_kernel<T, C>>(C::kSmemBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(teams * kGroup);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kGroup;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, mul_fp8_rows_kernel<T, C>, p, amap, bmap);
}

}  // namespace

size_t fp8_rows_scratch_bytes(int M, int N, int K, int sms) { return rows_bytes(plan_rows(M, N, K, sms)); }

cudaError_t launch_fp8_rows(const Fp8Args& a, int sms, cudaStream_t stream) {
  const RowsPlan plan = plan_rows(a.M, a.N, a.K, sms);
  RowsParams p;
  p.C = a.C;
  p.sa = a.sa;
  p.sb = a.sb;
  p.M = a.M;
  p.N = a.N;
  p.kb = a.kb;
  p.row_tiles = plan.row_tiles;
  p.tiles = plan.tiles;
  p.whole = plan.whole;
  p.extra = plan.extra;
  p.sharers = plan.sharers;
  p.weights_early = tc5_get_overlap() ? 1 : 0;
  p.arrived = static_cast<unsigned int*>(a.scratch) + kEpochWords;
  p.partials = reinterpret_cast<float4*>(static_cast<unsigned char*>(a.scratch) + kRowsScratch);
  p.status = a.status;
  CUtensorMap amap, bmap;
  cudaError_t e = encode_bytes_map(a.A, a.M, a.K, kBlock, &amap);
  if (e == cudaSuccess) e = encode_bytes_map(a.B, a.N, a.K, kBlock, &bmap);
  if (e != cudaSuccess) return e;
  if (plan.group == 1) return a.bf16 ? launch_rows<__nv_bfloat16, 1>(p, plan.teams, amap, bmap, stream) : launch_rows<half, 1>(p, plan.teams, amap, bmap, stream);
  return a.bf16 ? launch_rows<__nv_bfloat16, 2>(p, plan.teams, amap, bmap, stream) : launch_rows<half, 2>(p, plan.teams, amap, bmap, stream);
}

}  // namespace fp6m
