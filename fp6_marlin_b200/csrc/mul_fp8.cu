// C[m, n] = sum over blocks b of 128 values of K:  sa[m, b] * sb[n / 128, b] * sum_k A[m, k] * B[n, k]
//
// A (M x K) and B (N x K) in E4M3, fp32 scales, fp32 sums, C in fp16 or bf16 with one rounding.
// The reference has no counterpart: its weights have four or six bits.
//
// The product is computed transposed, as in the GEMMs of this library: 128 rows of B - one strip, and one scale per block of K -
// are the M dimension of tcgen05.mma.kind::f8f6f4 (a TMEM lane per column of C), up to 64 rows of A its N dimension (more: mul_fp8_rows.cu).  The scales
// change with every block of 128 values of K, so a block is one accumulator tile of its own (four MMAs, the first one overwrites):
// warps read it back, multiply it by sa * sb and add it to their sums in registers while the tensor cores work on the next blocks.
//
// Bound by the bytes of B.  8192 x 57344 (K x N), 16 rows, public calls one behind the other: 87.7 us, 5.4 TB/s, 0.82 of what a copy reaches; the rest is the first
// data of a CTA (about 4 us with the set-up) and the last ones' end.  4096 x 4096, one row: 7.6 us where the bytes take 2.6: set-up, first data, the exchange of sums.
// (Here and in the other kernel, figures of both sides of a choice are of replays of a graph.)
// The blocks are cut into as many ranges as there are multiprocessors, so a strip's sums mostly come from two or three CTAs: words of
// {value, tag} that the CTA in which the strip starts polls for; a tag needs no flag, no fence and no clearing.  A thread keeps at most 32 sums: with 64 of
// them (rows 65 to 192 in this form) they were spilled and 128 rows of 11008 x 4096 took 39 us, against 21 in the other kernel.
#include <limits.h>

#include "../../include/fp6m.h"
#include "host_common.h"
#include "mul_fp8.cuh"

namespace fp6m {

namespace {

struct Fp8Params {
  void* C;
  const float *sa, *sb;
  int M, N, kb;                          // kb: blocks of K
  int strips, tile_rows;                 // tile_rows: rows of A, rounded up to a multiple of 16
  int group_rows;                        // of them, those of a group of four warps; the last group may have fewer
  int weights_early;                     // the kernel in front does not write B: its first blocks are read before that has finished
  unsigned int* epochs;
  unsigned long long* partials;          // [CTA][tile_rows][128] words {value, tag}
  int* status;
};

template <int ROWS_, int WARPS_>
struct Fp8Cfg {
  static constexpr int kRows = ROWS_;                        // most rows of A per tile
  static constexpr int kWarps = WARPS_;                      // warps that read accumulators back, four share all 128 lanes
  static constexpr int kMine = kRows / (kWarps / 4);         // rows of a thread
  static constexpr int kStageBytes = kStripBytes + kRows * kBlock;
  static constexpr int kStages = 200 * 1024 / kStageBytes < 11 ? 200 * 1024 / kStageBytes : 11;
  static constexpr int kTiles = 4;       // accumulator tiles in tensor memory
  static constexpr int kTmemCols = kTiles * kRows < 32 ? 32 : kTiles * kRows;
  static constexpr int kScales = 8;                          // blocks whose scales wait in shared memory
  static constexpr int kNumBars = 2 * kStages + 2 * kTiles + 2 * kScales + 1;
  static constexpr int kThreads = 32 * (4 + kWarps);
  static constexpr int kOutRow = 32 * 2 + 16;                // bytes of a row of 32 finished values in shared memory, with a gap
  static constexpr int kSmemBytes = kStages * kStageBytes + kScales * kRows * 4 + kWarps * 16 * kOutRow + kNumBars * 8 + 16 + 1024;
  static constexpr int kChunk = kMine < 32 ? 16 : 32;     // values per read-back
};

// D[128 x N] = A[128 x 128] B[N x 128]^T of E4M3 values, both in 128-byte rows with the 128-byte swizzle: four MMAs of 32 values of K
__device__ __forceinline__ void mma_block(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(d_tmem), "l"(a_desc + 2 * i), "l"(b_desc + 2 * i), "r"(idesc), "r"(i) : "memory");
}
// The blocks of all strips, K fastest, are cut into as many equal ranges as there are CTAs.
__device__ __forceinline__ int range_start(const Fp8Params& p, int cta) {
  return (int)((long long)p.strips * p.kb * cta / (int)gridDim.x);
}

template <class T, class C>
__global__ void __launch_bounds__(C::kThreads, 1)
mul_fp8_kernel(const __grid_constant__ Fp8Params p, const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap) {
  constexpr int S = C::kStages, D = C::kTiles, R = C::kScales;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* scales = reinterpret_cast<float*>(smem + S * C::kStageBytes);
  uint8_t* out_stage = reinterpret_cast<uint8_t*>(scales + R * C::kRows);           // [warp][16 rows][kOutRow]
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_stage + C::kWarps * 16 * C::kOutRow);
  volatile uint32_t* misc = reinterpret_cast<uint32_t*>(bars + C::kNumBars);        // [0] TMEM base, [1] launch epoch
  const uint32_t full = smem_u32(bars), empty = full + 8 * S, done = empty + 8 * S, taken = done + 8 * D;
  const uint32_t scaled = taken + 8 * D, used = scaled + 8 * R, epoch_bar = used + 8 * R;

  const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31;
  // Ranges are handed out from the last to the first: a CTA that waits for the partials of higher ranges waits for CTAs that
  // were dispatched before it.
  const int cta = gridDim.x - 1 - blockIdx.x;
  const int B0 = range_start(p, cta), B1 = range_start(p, cta + 1);
  const int nt = p.tile_rows;
  launch_dependents();

  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full + 8 * s, 1);            // the expect_tx arrival of the producer
      mbar_init(empty + 8 * s, 1);           // tcgen05.commit: the block's MMAs have read the stage
    }
    for (int d = 0; d < D; ++d) {
      mbar_init(done + 8 * d, 1);            // tcgen05.commit: the tile holds the block's products
      mbar_init(taken + 8 * d, C::kWarps);   // the warps have read it back
    }
    for (int r = 0; r < R; ++r) {
      mbar_init(scaled + 8 * r, 1);
      mbar_init(used + 8 * r, C::kWarps);
    }
    mbar_init(epoch_bar, 1);
    mbar_fence_init();
  }
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(misc))), "r"(C::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, misc[0], 0);
  bool dead = false;

  if (warp == 0) {
    // ================================================================== producer of weights and activations
    const uint32_t bytes = kStripBytes + nt * kBlock;
    const int first = B1 - B0 < S ? B1 - B0 : S;                     // blocks whose stages are free from the start
    // (places are counted on: divisions by run-time values would take longer than a block)
    struct Place {
      int x, row;                                                    // byte of K, row of B
    };
    const Place start = {B0 % p.kb * kBlock, B0 / p.kb * kBlock};
    auto next = [&](Place& at) {
      at.x += kBlock;
      if (at.x < p.kb * kBlock) return;
      at.x = 0;
      at.row += kBlock;
    };
    auto load_weights = [&](int n, const Place& at) {
      mbar_arrive_expect_tx(full + 8 * n, bytes);
      tma_load_bytes(smem_u32(smem) + n * C::kStageBytes, &bmap, at.x, at.row, full + 8 * n);
    };
    auto load_rows = [&](int n, const Place& at) {
      tma_load_bytes(smem_u32(smem) + n * C::kStageBytes + kStripBytes, &amap, at.x, 0, full + 8 * n);
    };
    Place at = start;
    for (int n = 0; n < first; ++n) {
      if (elect_one()) {
        if (p.weights_early) load_weights(n, at);
        else tma_prefetch_bytes(&bmap, at.x, at.row);
      }
      next(at);
    }
    __syncwarp();
    grid_dependency_wait();
    at = start;
    for (int n = 0; n < first; ++n) {
      if (elect_one()) {
        if (!p.weights_early) load_weights(n, at);
        load_rows(n, at);
      }
      next(at);
    }
    __syncwarp();
    int stage = 0;
    uint32_t phase = 0;
    for (int u = B0 + first; u < B1; ++u) {
      mbar_wait_bounded<100>(empty + 8 * stage, phase, p.status, dead);
      if (elect_one()) {
        load_weights(stage, at);
        load_rows(stage, at);
      }
      __syncwarp();
      next(at);
      if (++stage == S) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    // ================================================================== MMA issuer
    grid_dependency_wait();                  // the bounded waits start when the kernel in front has finished
    const uint64_t desc0 = wide_act_desc(smem_u32(smem));
    // D fp32, A and B E4M3, K-major; N = rows of the tile, M = 128
    const uint32_t idesc = (1u << 4) | ((uint32_t)(nt >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    int stage = 0, tile = 0;
    uint32_t phase = 0, tphase = 0;
    for (int u = B0; u < B1; ++u) {
      mbar_wait_bounded<20>(taken + 8 * tile, tphase ^ 1, p.status, dead);
      mbar_wait_bounded<20>(full + 8 * stage, phase, p.status, dead);
      tc_fence_after();
      // the descriptor's low 14 bits hold the address / 16: adding an offset never carries out of them
      const uint64_t a_desc = desc0 + (uint64_t)(stage * (C::kStageBytes >> 4));
      if (elect_one()) {
        mma_block(tmem + tile * C::kRows, a_desc, a_desc + (kStripBytes >> 4), idesc);
        tc_commit(empty + 8 * stage);
        tc_commit(done + 8 * tile);
      }
      __syncwarp();
      if (++stage == S) { stage = 0; phase ^= 1; }
      if (++tile == D) { tile = 0; tphase ^= 1; }
    }
  } else if (warp == 2) {
    // ================================================================== scales: sa * sb of the block for every row of the tile
    grid_dependency_wait();
    // The scales of kAhead blocks are on their way together: with one block at a time the loads' latency was longer than a block takes.
    constexpr int E = (C::kRows + 31) / 32, kAhead = 4;
    float now[kAhead][E], column[kAhead];
    int b = B0 % p.kb, strip = B0 / p.kb, left = B1 - B0;      // of the block to load
    auto load = [&](int j) {
      const bool live = left > 0;
      column[j] = live ? p.sb[(size_t)strip * p.kb + b] : 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int m = lane + 32 * i;
        now[j][i] = live && m < p.M ? p.sa[(size_t)m * p.kb + b] : 0.f;
      }
      --left;
      if (++b == p.kb) {
        b = 0;
        ++strip;
      }
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(j);
    int r = 0;
    uint32_t phase = 0;
    for (int u0 = B0; u0 < B1; u0 += kAhead) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (u0 + j >= B1) break;
        mbar_wait_bounded<100>(used + 8 * r, phase ^ 1, p.status, dead);
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (C::kRows % 32 == 0 || lane + 32 * i < C::kRows) sts_f32(smem_u32(scales + r * C::kRows + lane + 32 * i), now[j][i] * column[j]);
        __syncwarp();
        if (lane == 0) mbar_arrive(scaled + 8 * r);
        load(j);
        if (++r == R) { r = 0; phase ^= 1; }
      }
    }
  } else if (warp == 3) {
    // ================================================================== launch epoch: the tag of this launch's partials is epoch + 1
    if (lane == 0) {
      grid_dependency_wait();
      misc[1] = read_epoch_and_count(p.epochs, gridDim.x);
      mbar_arrive(epoch_bar);
    }
    __syncwarp();
  } else {
    // ================================================================== sums: thread = column of the strip, kMine rows
    constexpr int CH = C::kChunk, E = C::kMine;
    const int quarter = warp & 3, row_base = (warp - 4) / 4 * p.group_rows;
    const int c = quarter * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + row_base;
    const int my_rows = min(p.group_rows, nt - row_base);
    grid_dependency_wait();
    float sum[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = 0.f;
    int tile = 0, r = 0, slice_start = B0, block = B0 % p.kb;
    uint32_t tphase = 0, rphase = 0;
    for (int u = B0; u < B1; ++u) {
      mbar_wait_bounded<20>(scaled + 8 * r, rphase, p.status, dead);
      mbar_wait_bounded<20>(done + 8 * tile, tphase, p.status, dead);
      tc_fence_after();
      // all read-backs are on their way before the scales are loaded, and the tile is given back before the sums
      uint32_t v[E];
#pragma unroll
      for (int c0 = 0; c0 < E; c0 += CH)
        if (c0 < my_rows) tmem_load<CH>(lane_base + tile * C::kRows + c0, v + c0);       // the same for all threads of the warp
      const uint32_t from = smem_u32(scales + r * C::kRows + row_base);
      float4 scale[E / 4];
#pragma unroll
      for (int i = 0; i < E / 4; ++i) scale[i] = lds_float4(from + 16 * i);
      tmem_loaded<E>(v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(taken + 8 * tile);
        mbar_arrive(used + 8 * r);
      }
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        sum[4 * i] = fmaf(__uint_as_float(v[4 * i]), scale[i].x, sum[4 * i]);
        sum[4 * i + 1] = fmaf(__uint_as_float(v[4 * i + 1]), scale[i].y, sum[4 * i + 1]);
        sum[4 * i + 2] = fmaf(__uint_as_float(v[4 * i + 2]), scale[i].z, sum[4 * i + 2]);
        sum[4 * i + 3] = fmaf(__uint_as_float(v[4 * i + 3]), scale[i].w, sum[4 * i + 3]);
      }
      if (++tile == D) { tile = 0; tphase ^= 1; }
      if (++r == R) { r = 0; rphase ^= 1; }

      const bool strip_ends = ++block == p.kb;
      if (strip_ends) block = 0;
      if (!strip_ends && u + 1 < B1) continue;
      // ---- the end of a slice: this CTA's blocks of one strip
      const int strip = u / p.kb, column = strip * kBlock + c;
      const bool starts = slice_start % p.kb == 0;
      const int rows = min(my_rows, p.M - row_base);           // rows of this thread that exist
      uint32_t tag = 0;
      if (!starts || !strip_ends) {
        mbar_wait_bounded<20>(epoch_bar, 0, p.status, dead);
        tag = misc[1] + 1;
      }
      auto slot_of = [&](int other) { return p.partials + ((size_t)other * nt + row_base) * kBlock + c; };
      if (!starts) {
        // Only the first slice of a CTA can start inside a strip, so a CTA has one partial.
        unsigned long long* slot = slot_of(cta);
        each<0, E>([&](auto i) {
          if (i < rows) st_partial<i * kBlock>(slot, ((unsigned long long)tag << 32) | __float_as_uint(sum[i]));
        });
      } else {
        // The CTA in which a strip starts adds the partials of the CTAs behind it, in their order.
        if (!strip_ends) {
          const int end = (strip + 1) * p.kb;
#pragma unroll 1
          for (int other = cta + 1; other < (int)gridDim.x && range_start(p, other) < end; ++other) {
            const unsigned long long* slot = slot_of(other);
            each<0, E / 16>([&](auto part) {
              constexpr int i0 = 16 * part;
              if (i0 >= rows) return;
              unsigned long long w[16];
              bool here = false;
#pragma unroll 1
              for (int spin = 0; spin < (1 << 20) && !here; ++spin) {
                each<0, 16>([&](auto i) { w[i] = i0 + i < rows ? ld_partial<(i0 + i) * kBlock>(slot) : (unsigned long long)tag << 32; });
                here = true;
#pragma unroll
                for (int i = 0; i < 16; ++i) here = here && (uint32_t)(w[i] >> 32) == tag;
                if (dead) break;             // a wait of this thread ran out before: do not wait again
              }
              if (!here && !dead) {
                dead = true;
                if (p.status) atomicExch(p.status, kStatusTimeout);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) sum[i0 + i] += __uint_as_float((uint32_t)w[i]);
            });
          }
        }
        // A warp turns 16 rows x 32 columns at a time round in shared memory and stores sixteen bytes a lane.
        uint8_t* mine = out_stage + (warp - 4) * 16 * C::kOutRow;
        const int out_column = column - lane + (lane & 3) * 8;
#pragma unroll
        for (int i0 = 0; i0 < E; i0 += 16) {
          if (i0 >= rows) break;
#pragma unroll
          for (int i = 0; i < 16; ++i) store_value(reinterpret_cast<T*>(mine + i * C::kOutRow) + lane, sum[i0 + i]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            const int r = i + (lane >> 2);
            if (i0 + r < rows && out_column < p.N)
              *reinterpret_cast<uint4*>(static_cast<T*>(p.C) + (size_t)(row_base + i0 + r) * p.N + out_column) = *reinterpret_cast<const uint4*>(mine + r * C::kOutRow + (lane & 3) * 16);
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int i = 0; i < E; ++i) sum[i] = 0.f;
      slice_start = u + 1;
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
}

// The kernels' places are of 32 bits, also those of the last tile's end.
bool fp8_sizes_fit(int M, int N, int K) { return M <= INT_MAX - 255 && N <= INT_MAX - 255 && K <= INT_MAX - 255; }
int columns_ctas(int N, int K, int sms) {
  const long long blocks = (long long)((N + kBlock - 1) / kBlock) * ((K + kBlock - 1) / kBlock);
  const int ctas = sms > 0 && sms < kMaxFp8Ctas ? sms : kMaxFp8Ctas;
  // (at least four blocks each: fewer take less time than joining what more CTAs leave)
  return ctas < (blocks + 3) / 4 ? ctas : (int)((blocks + 3) / 4);
}
size_t columns_scratch_bytes(int M, int N, int K, int sms) {
  return kFp8Header + (size_t)columns_ctas(N, K, sms) * ((M + 15) / 16 * 16) * kBlock * sizeof(unsigned long long);
}
size_t fp8_scratch_bytes(int M, int N, int K, int sms) {
  return M <= kMostColumnsRows ? columns_scratch_bytes(M, N, K, sms) : fp8_rows_scratch_bytes(M, N, K, sms);
}

template <class T, class C>
cudaError_t launch_with(const Fp8Params& p, int ctas, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  cudaError_t e = allow_shared_memory<mul_fp8_kernel<T, C>>(C::kSmemBytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(mul_fp8_kernel<T, C>, dim3(ctas), dim3(C::kThreads), C::kSmemBytes, stream, p, amap, bmap);
}
template <class T>
cudaError_t launch_typed(const Fp8Params& p, int ctas, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  if (p.tile_rows <= 16) return launch_with<T, Fp8Cfg<16, 4>>(p, ctas, amap, bmap, stream);
  if (p.tile_rows <= 32) return launch_with<T, Fp8Cfg<32, 4>>(p, ctas, amap, bmap, stream);
  return launch_with<T, Fp8Cfg<64, 8>>(p, ctas, amap, bmap, stream);
}
cudaError_t launch_fp8_columns(const Fp8Args& a, int sms, cudaStream_t stream) {
  Fp8Params p;
  p.C = a.C;
  p.sa = a.sa;
  p.sb = a.sb;
  p.M = a.M;
  p.N = a.N;
  p.kb = a.kb;
  p.strips = (a.N + kBlock - 1) / kBlock;
  p.tile_rows = (a.M + 15) / 16 * 16;
  p.group_rows = p.tile_rows <= 32 ? p.tile_rows : 32;
  p.weights_early = tc5_get_overlap() ? 1 : 0;
  p.epochs = static_cast<unsigned int*>(a.scratch);
  p.partials = reinterpret_cast<unsigned long long*>(static_cast<unsigned char*>(a.scratch) + kFp8Header);
  p.status = a.status;
  CUtensorMap amap, bmap;
  cudaError_t e = encode_bytes_map(a.A, a.M, a.K, p.tile_rows, &amap);
  if (e == cudaSuccess) e = encode_bytes_map(a.B, a.N, a.K, kBlock, &bmap);
  if (e != cudaSuccess) return e;
  const int ctas = columns_ctas(a.N, a.K, sms);
  return a.bf16 ? launch_typed<__nv_bfloat16>(p, ctas, amap, bmap, stream) : launch_typed<half>(p, ctas, amap, bmap, stream);
}

}  // namespace

}  // namespace fp6m

extern "C" {

size_t fp6m_mul_fp8_scratch_bytes(int M, int N, int K, int sms) {
  if (M <= 0 || N <= 0 || K <= 0 || !fp6m::fp8_sizes_fit(M, N, K)) return 256;
  return (fp6m::fp8_scratch_bytes(M, N, K, sms) + 255) & ~(size_t)255;
}

int fp6m_mul_fp8(const void* A, const void* B, void* C, const void* sa, const void* sb, int M, int N, int K, int type, void* scratch, size_t scratch_bytes,
                 int dev, void* stream, int* status_dev) {
  using namespace fp6m;
  if (M < 0 || N < 0 || K < 0 || (type != FP6M_TYPE_F16 && type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (K % 16 || N % 8 || !fp8_sizes_fit(M, N, K)) return FP6M_ERR_PROB_SHAPE;
  if (M == 0 || N == 0) return FP6M_OK;
  if (!C || !aligned16(C)) return FP6M_ERR_BAD_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) {                          // an empty sum
    DeviceGuard guard(dev);
    const cudaError_t e = cudaMemsetAsync(C, 0, (size_t)M * N * 2, st);
    return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "mul_fp8 of no terms");
  }
  if (!A || !B || !sa || !sb || !scratch || !aligned16(A) || !aligned16(B) || !aligned16(scratch) ||
      ((reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sb)) & 3))
    return FP6M_ERR_BAD_ARG;
  if ((long long)((N + kBlock - 1) / kBlock) * ((M + 127) / 128) * ((K + kBlock - 1) / kBlock) > 0x3fffffff) return FP6M_ERR_PROB_SHAPE;
  DeviceGuard guard(dev);
  const int sms = sm_count(dev);
  if (sms <= 0) return cuda_fail(cudaGetLastError(), "cudaDeviceGetAttribute");
  if (scratch_bytes < fp8_scratch_bytes(M, N, K, sms)) return FP6M_ERR_SCRATCH;
  const Fp8Args a = {A, B, C, static_cast<const float*>(sa), static_cast<const float*>(sb), M, N, K, (K + kBlock - 1) / kBlock, type == FP6M_TYPE_BF16, scratch, status_dev};
  const cudaError_t e = M <= kMostColumnsRows ? launch_fp8_columns(a, sms, st) : launch_fp8_rows(a, sms, st);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "mul_fp8 launch");
}

}  // extern "C"
