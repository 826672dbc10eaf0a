// C = A B^T of E4M3 matrices with scales for blocks of 128, more than 64 rows of A: see mul_fp8.cu for the product itself.
//
// Here the rows of A are the lanes of the accumulators: a thread sums columns of one row of C, so a block of K has one scale per
// thread - sa of its row times sb of its columns - and not one per value.  More than 128 rows: two CTAs share a tile of 256 rows
// and 256 columns (cta_group::2).  Each brings 128 rows of A and half of the columns of B, 32 KB per block of K for 512 cycles of
// the tensor cores; one CTA alone would have to bring 48 KB, more than the 64 bytes a cycle that reach a multiprocessor.
// Up to 128 rows: one CTA, 128 columns.
//
// Every pair of CTAs (or CTA) computes whole tiles, in the order of the tiles, as long as all have one; what is left is cut along K
// into equal ranges, whose sums are exchanged as in mul_fp8.cu.
#include "../../include/fp6m.h"
#include "host_common.h"
#include "mul_fp8.cuh"

namespace fp6m {

namespace {

constexpr int kMaxTeams = 192;

struct RowsParams {
  void* C;
  const float *sa, *sb;
  int M, N, kb;
  int row_tiles, tiles;                  // tiles in the order of their columns, row tiles next to one another
  int whole;                             // whole tiles of every team
  int sharers;                           // teams that share the tiles that are left, cut along K
  int weights_early;
  unsigned int* epochs;
  unsigned long long* partials;          // [CTA][value][thread] words {value, tag}
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
  static constexpr int kNumBars = 2 * kStages + 2 * kTiles + 1;
  static constexpr int kOutRow = 32 * 2 + 16;                // bytes of a row of 32 finished values in shared memory, with a gap
  static constexpr int kSmemBytes = kStages * kStageBytes + kWarps * 32 * kOutRow + kNumBars * 8 + 16 + 1024;
  static constexpr int kSlotWords = kMine * kWarps * 32;
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
    return (long long)(p.tiles - p.whole * teams) * p.kb * min(team, p.sharers) / max(p.sharers, 1);
  }
  __device__ __forceinline__ long long start_of(const RowsParams& p, int t) const { return start_of(p, t, teams); }
  __device__ __forceinline__ bool next(const RowsParams& p, int& tile, int& k0, int& k1) {
    if (index < p.whole) {
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
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
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
// two sums at a time
__device__ __forceinline__ void fma2(unsigned long long& sum, uint32_t lo, uint32_t hi, unsigned long long scale) {
  asm("{\n.reg .b64 v;\nmov.b64 v, {%1, %2};\nfma.rn.f32x2 %0, v, %3, %0;\n}\n" : "+l"(sum) : "r"(lo), "r"(hi), "l"(scale));
}
__device__ __forceinline__ float low(unsigned long long v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high(unsigned long long v) { return __uint_as_float((uint32_t)(v >> 32)); }

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
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_stage + C::kWarps * 32 * C::kOutRow);
  volatile uint32_t* misc = reinterpret_cast<uint32_t*>(bars + C::kNumBars);        // [0] TMEM base, [1] launch epoch
  const uint32_t full = smem_u32(bars), empty = full + 8 * S, done = empty + 8 * S, taken = done + 8 * D, epoch_bar = taken + 8 * D;

  const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31;
  const int rank = G == 1 ? 0 : blockIdx.x & 1;              // in the team (clusters are neighbouring CTAs)
  // Ranges are handed out from the last to the first: a team that waits for the partials of higher ones waits for CTAs that were
  // dispatched before it.
  const int teams = gridDim.x / G, team = teams - 1 - (int)blockIdx.x / G;
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
    mbar_init(epoch_bar, 1);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    grid_dependency_wait();
  } else if (warp == 3) {
    // ================================================================== launch epoch: the tag of this launch's partials is epoch + 1
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (lane == 0) {
      grid_dependency_wait();
      misc[1] = read_epoch_and_count(p.epochs, gridDim.x);
      mbar_arrive(epoch_bar);
    }
    __syncwarp();
  } else {
    // ================================================================== sums: thread = row of the tile, kMine columns
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    constexpr int E = C::kMine;
    const int quarter = warp & 3, half_index = (warp - 4) >> 2;
    const int row_in = quarter * 32 + lane, column_in = half_index * E;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + column_in;
    const uint32_t taken0 = G == 1 ? taken : in_leader(taken);
    grid_dependency_wait();
    unsigned long long sum[E / 2];                           // pairs of fp32 sums
    int buffer = 0;
    uint32_t tphase = 0;
    float now[4], coming[4], coming_sb[4];                   // scales of four blocks, and of the next four, which are multiplied when they are used
    const float *sa = nullptr, *sb = nullptr;
    bool row_lives = false;
    auto open = [&](int tile) {
      const int row = tile % p.row_tiles * (128 * G) + rank * 128 + row_in;
      const int block = ((tile / p.row_tiles) * C::kColumns + column_in) / kBlock;
      row_lives = row < p.M;
      sa = p.sa + (size_t)(row_lives ? row : 0) * p.kb;
      sb = p.sb + (size_t)min(block, (p.N - 1) / kBlock) * p.kb;
    };
    auto fetch = [&](int k, int k1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        coming[j] = row_lives && k + j < k1 ? sa[k + j] : 0.f;
        coming_sb[j] = k + j < k1 ? sb[k + j] : 0.f;
      }
    };
    bool more = segments.next(p, tile, k0, k1);
    if (more) {
      open(tile);
      fetch(k0, k1);
    }
    while (more) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) sum[i] = 0;
      for (int k = k0; k < k1; k += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) now[j] = coming[j] * coming_sb[j];
        fetch(k + 4, k1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (k + j >= k1) break;
          unsigned long long scale;
          asm("mov.b64 %0, {%1, %1};" : "=l"(scale) : "f"(now[j]));
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
            for (int i = 0; i < 16; ++i) fma2(sum[c * 16 + i], v[c & 1][2 * i], v[c & 1][2 * i + 1], scale);
          }
          if (++buffer == D) { buffer = 0; tphase ^= 1; }
        }
      }
      // ---- the end of a segment
      const int row0 = tile % p.row_tiles * (128 * G) + rank * 128 + quarter * 32, column0 = (tile / p.row_tiles) * C::kColumns + column_in;
      const bool starts = k0 == 0, ends = k1 == p.kb;
      const int shared_tile = tile - p.whole * teams;
      more = segments.next(p, tile, k0, k1);
      if (more) {                                            // the next segment's first scales
        open(tile);
        fetch(k0, k1);
      }
      uint32_t tag = 0;
      if (!starts || !ends) {
        mbar_wait_bounded<20>(epoch_bar, 0, p.status, dead);
        tag = misc[1] + 1;
      }
      auto slot_of = [&](int other) { return p.partials + (size_t)(other * G + rank) * C::kSlotWords + (warp - 4) * 32 + lane; };
      constexpr int kStep = C::kWarps * 32;
      if (!starts) {
        // only a team's first segment of the shared tiles can start inside a tile, so a CTA has one partial
        unsigned long long* slot = slot_of(team);
        each<0, E / 2>([&](auto i) {
          st_partial<2 * i * kStep>(slot, ((unsigned long long)tag << 32) | (uint32_t)sum[i]);
          st_partial<(2 * i + 1) * kStep>(slot, ((unsigned long long)tag << 32) | (sum[i] >> 32));
        });
        continue;
      }
      if (!ends) {
        // The team in which a tile starts adds the partials of the teams behind it, in their order.
        const long long end = (long long)(shared_tile + 1) * p.kb;
#pragma unroll 1
        for (int other = team + 1; other < teams && segments.start_of(p, other) < end; ++other) {
          if (segments.start_of(p, other) >= segments.start_of(p, other + 1)) break;
          const unsigned long long* slot = slot_of(other);
          each<0, E / 16>([&](auto part) {
            constexpr int i0 = 16 * part;
            unsigned long long w[16];
            bool here = false;
#pragma unroll 1
            for (int spin = 0; spin < (1 << 20) && !here; ++spin) {
              each<0, 16>([&](auto i) { w[i] = ld_partial<(i0 + i) * kStep>(slot); });
              here = true;
#pragma unroll
              for (int i = 0; i < 16; ++i) here = here && (uint32_t)(w[i] >> 32) == tag;
              if (dead) break;                               // a wait of this thread ran out before: do not wait again
            }
            if (!here && !dead) {
              dead = true;
              if (p.status) atomicExch(p.status, kStatusTimeout);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const unsigned long long two = (w[2 * i] & 0xffffffffull) | w[2 * i + 1] << 32;
              asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[i0 / 2 + i]) : "l"(two));
            }
          });
        }
      }
      // A warp turns 32 rows x 32 columns at a time round in shared memory: four lanes store 64 bytes of a row.
      uint8_t* mine = out_stage + (warp - 4) * 32 * C::kOutRow;
#pragma unroll
      for (int c = 0; c < E / 32; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = Two<T>::pack(low(sum[c * 16 + i * 4 + e]), high(sum[c * 16 + i * 4 + e]));
          *reinterpret_cast<uint4*>(mine + lane * C::kOutRow + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        const int column = column0 + c * 32 + (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 2);
          if (row0 + r < p.M && column < p.N)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.C) + (size_t)(row0 + r) * p.N + column) = *reinterpret_cast<const uint4*>(mine + r * C::kOutRow + (lane & 3) * 16);
        }
        __syncwarp();
      }
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
  int group, row_tiles, tiles, teams, whole, sharers;
};
RowsPlan plan_rows(int M, int N, int K, int sms) {
  RowsPlan plan;
  plan.group = M <= 128 ? 1 : 2;
  const int edge = 128 * plan.group, kb = (K + kBlock - 1) / kBlock;
  plan.row_tiles = (M + edge - 1) / edge;
  plan.tiles = plan.row_tiles * ((N + edge - 1) / edge);
  int teams = (sms > 0 && sms < kMaxTeams ? sms : kMaxTeams) / plan.group;
  const long long blocks = (long long)plan.tiles * kb;
  if (teams > (blocks + 3) / 4) teams = (int)((blocks + 3) / 4);
  plan.teams = teams < 1 ? 1 : teams;
  plan.whole = plan.tiles / plan.teams;
  const long long left = (long long)(plan.tiles - plan.whole * plan.teams) * kb;
  plan.sharers = (int)(left / 4 < plan.teams ? (left + 3) / 4 : plan.teams);
  return plan;
}
size_t rows_bytes(const RowsPlan& plan) {
  return kEpochWords * sizeof(unsigned int) + (size_t)plan.teams * plan.group * (plan.group * 64) * 256 * sizeof(unsigned long long);
}

template <class T, int kGroup>
cudaError_t launch_rows(const RowsParams& p, int teams, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  using C = RowsCfg<kGroup>;
  static_assert(C::kSlotWords == kGroup * 64 * 256, "slot");
  cudaError_t e = cudaFuncSetAttribute(mul_fp8_rows_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
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
  p.sharers = plan.sharers;
  p.weights_early = tc5_get_overlap() ? 1 : 0;
  p.epochs = static_cast<unsigned int*>(a.scratch);
  p.partials = reinterpret_cast<unsigned long long*>(static_cast<unsigned char*>(a.scratch) + kEpochWords * sizeof(unsigned int));
  p.status = a.status;
  CUtensorMap amap, bmap;
  cudaError_t e = encode_bytes_map(a.A, a.M, a.K, kBlock, &amap);
  if (e == cudaSuccess) e = encode_bytes_map(a.B, a.N, a.K, kBlock, &bmap);
  if (e != cudaSuccess) return e;
  if (plan.group == 1) return a.bf16 ? launch_rows<__nv_bfloat16, 1>(p, plan.teams, amap, bmap, stream) : launch_rows<half, 1>(p, plan.teams, amap, bmap, stream);
  return a.bf16 ? launch_rows<__nv_bfloat16, 2>(p, plan.teams, amap, bmap, stream) : launch_rows<half, 2>(p, plan.teams, amap, bmap, stream);
}

}  // namespace fp6m
