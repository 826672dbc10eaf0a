// Attention of drafted tokens over a paged cache in 8 bits: as tree_attention.cu, but committed keys and values are E4M3 with a power of two for each
// token and head (cache_fp8.cu writes them).
//
//   k_j = 2^x_j * K_j,  v_j = 2^y_j * V_j     K_j, V_j in E4M3, exact in fp16
//   a_ij = scale * log2(e) * 2^x_j * (q_i . K_j) + y_j,   M_i = max_j a_ij,   w_ij = 2^(a_ij - M_i)
//   o_i  = sum_j w_ij V_j / sum_j 2^-y_j w_ij
//
// so that the scales cost one fused multiply-add per score and none per key or value: the values' power is an addend of the exponent, and the maximum that
// keeps the exponentials in range is that of the weights as they meet the values.  These are rounded once, to fp16 (2^-11 of a weight; below 2^-14 of the largest they
// become multiples of 2^-24), for both types of queries; the sum that they are divided by has them unrounded, 2^-y_j w_ij = 2^(a_ij - M_i - y_j) as an exponential of its own:
// a w_ij that is zero beside those of values 2^150 times larger may be most of the sum.  Its terms come times 2^40, so that fp32 holds them for powers of values from 2^-54 (the largest
// term is below 2^(8 + 54 + 40)) to 2^120 (the largest is not below 2^(40 - 120), and what is below 2^-126 counts nothing).  Queries in bf16 come as fp16 times a power of
// two for each row, with the largest value between 2^14 and 2^15: exact but for values 2^-28 times smaller than that.
//
// Drafted keys and values are 16 bits.  They make a tile of their own behind the cached ones, which is brought into the form of the others when it is worked
// on: fp16 with a power of two per token (bf16 as the queries, values with 2^-54 at least; fp16 as it is).
//
// Work is cut into equal ranges of (sequence, head of keys, row tile, key tile) units as in tree_attention.cu.
//
// Products are transposed, so that a step of mma.sync covers 16 tokens and 8 rows and what is converted to fp16 - sixteen tokens' keys or values, a
// warp's share of a tile - serves all rows:   S^T (tokens x rows) = K Q^T,   O^T (values x rows) += V^T W^T.   With a thread's four neighbouring E4M3 values as the pairs that
// the two halves of a step's operand want, queries are permuted alike and nothing is shuffled; values are transposed by ldmatrix in pairs and come apart into even and odd ones.
// One warp copies (runs of a page by TMA, else sixteen bytes a thread), one brings the tokens' powers of two, four compute; nothing but a stage's two barriers is between them.
//
// mma.sync and not tcgen05: E4M3 times E4M3 is not wanted (queries and weights keep 11 bits), so keys and values pass through registers in any case, and at up to 32 rows the tensor pipe is
// busy a sixth (one row) to a third (32) of the time.  32 rows take less here than there: see kFewRows.
//
// Up to 8 rows bound by the copies: the same kernel with no arithmetic at all takes as long (issue slots are busy 42 % of the time, the pipe of the conversions 44 %).  More rows: by the
// chains of the four computing warps, whose tiles follow one another through products, maxima, exponentials and products; no unit is busy half of the time (32 rows: issue slots 45 %, conversions 41 %,
// tensor pipe 31 %, special functions 17 %, memory 32 %).  Replays of a graph, heads of 128:
//   64 x 1 token, 64 heads over 8, up to 8192    101 to 104 us, 5.2 TB/s, 0.79 of what a copy reaches; without joins 101; with a cache that lies head by head 98 to 101
//   64 x 1 / 2 / 3 / 4 (8 to 32 rows), 6144      82 / 106 / 152 / 155 us in bf16, 79 / 100 / 146 / 149 in fp16
//   3 x 1, 32 over 4, 65537                      43 us, 0.72; without joins 38
//   8 x 5, 32 over 32, up to 4096                33.4 us, 0.62; without joins 31
//   1 x 1, 32 over 32, 300                       8.6 us, without arithmetic 7.3: plan, look-ups, queries, first data, tiles and a join, one after the other
#include <cuda.h>

#include <type_traits>

#include "device_utils.cuh"
#include "gemm_params.h"
#include "host_common.h"
#include "tree_attention.cuh"

namespace {

using namespace fp6m;

constexpr int kWorkers = 128, kThreads = kWorkers + 64;
constexpr int kTile = 64, kDrafted = 32;           // cached tokens of a tile; places for drafted ones in theirs
constexpr int kRowTile = kFewRows;
constexpr int kLeastPower = -54, kTotalPower = 40; // of values; of what a row's total is kept times
// See make_plan.  us in graph replays with a slack of 4 / 8 / 16 / 32: one token over 300, 32 heads 10.1 / 8.5 / 8.5 / 8.6; sixteen over up to 500, 32 over 8 11.7 / 11.6 / 10.7 / 10.8; one
// over 1000, 32 over 8 10.1 / 9.9 / 10.1 / 14.4.  With at least 3 / 4 / 6 units per CTA: the last one 9.6 / 10.1 / 14.6, twice eight tokens over 2000 21.9 / 21.2 /
// 23.4; over 8192, 64 heads over 8, four tokens 29.7 / 27.0 / 27.9, two 22.0 / 20.5 / 20.7, one 15.5 / 14.7 / 15.0.  With rows taken to cost 2 / 4 / 7 tiles: 8 x 5 tokens, 32 heads, up to 4096 42.8 / 34.1 / 34.3.
constexpr int kLeastUnits = 4, kSlack = 16;

struct Fp8Params : TreeParams {
  int grain;                             // tokens of a page that start at a multiple of their number in a tile
  fp6m_cache_scales scales;
};

// A partial: sums [row][value], maxima, totals.  A CTA has three: of an item that it does not start, of one that it starts, of a group (see join_step).
template <int D>
constexpr int slot_floats() { return kRowTile * (D + 2); }
constexpr int kSlots = 3;

// Tiles of cached tokens, then one of the drafted tokens.
struct TilesApart {
  static __device__ __forceinline__ int of(const TreeParams&, int length) { return (length + kTile - 1) / kTile + 1; }
};
using Ranges = SegmentsOf<TilesApart>;

// NT: groups of eight rows that a warp works on; RW: warps that share the rows of an item (the others share the tokens of a tile).
template <int D, int NT, int RW>
struct Cfg {
  static constexpr int kGroups = NT * RW;
  static constexpr int kCtas = 2;                                    // per multiprocessor
  static constexpr int kKeyWarps = 4 / RW, kTogether = 2 / RW;       // a warp works on 32 tokens at a time, sixteen of two tiles or 32 of one
  static constexpr int kTileBytes = kTile * D, kStageBytes = 2 * kTileBytes;     // keys or values of a tile
  static constexpr int kStages = 5 * 128 / D;
  static constexpr int kPoolRow = D + 8;                             // floats, so that rows start in different banks
  static constexpr int kPowers = kStages * kStageBytes;              // uint32_t [stage][keys, values][kTile]: words with a token's exponent
  static constexpr int kWhere = kPowers + kStages * kTile * 8;       // uint32_t [stage][kTile]: where in these words
  static constexpr int kPool = kWhere + kStages * kTile * 4;         // float [warp][8][kPoolRow]
  static constexpr int kStats = kPool + 4 * 8 * kPoolRow * 4;        // float2 [warp][8 NT]: maximum, total
  static constexpr int kMasks = kStats + 4 * 8 * NT * 8;             // [8 kGroups]
  static constexpr int kBars = kMasks + 8 * kGroups * 8;
  static constexpr int kPlan = kBars + 2 * kStages * 8;
  // Queries: in registers where there is one group, else uint2 [D / 16][kGroups][32] and float [8 kGroups].  (What does not fit the 168 registers of a thread goes through the little that
  // shared memory leaves of L1: with 100 to 800 bytes of it, steps of 16 and 32 rows took 3900 and 6900 cycles.)
  static constexpr bool kSharedQueries = NT > 1;
  static constexpr int kQueries = (kPlan + (int)sizeof(Plan) + 15) / 16 * 16;
  static constexpr int kBytes = kQueries + (kSharedQueries ? D / 16 * kGroups * 32 * 8 + 8 * kGroups * 4 : 0) + 1024;
  static_assert(kCtas * (kBytes + 1024) <= 233472, "shared memory");
};

// an 8 x 8 matrix of 16-bit values, two neighbours of a row a thread: transposed
__device__ __forceinline__ uint32_t transposed(uint32_t m) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(m));
  return t;
}
// 2^n, -127 <= n <= 128
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float(n > -127 ? (uint32_t)(n + 127) << 23 : 0x00400000u); }
// the exponent that brings values of up to `top` below 2^15: fp16 holds them and what is up to 2^29 times smaller
__device__ __forceinline__ int exponent_for_half(float top) { return top == 0.f ? 0 : max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100); }
__device__ __forceinline__ float finite_magnitude(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
template <class T>
__device__ __forceinline__ float largest_of(uint32_t two) { return fmaxf(finite_magnitude(Half16<T>::value((uint16_t)two)), finite_magnitude(Half16<T>::value((uint16_t)(two >> 16)))); }
template <class T>
__device__ __forceinline__ uint32_t scaled_halves(uint32_t two, float by) { return Half16<half>::pack(Half16<T>::value((uint16_t)two) * by, Half16<T>::value((uint16_t)(two >> 16)) * by); }

// A total that is kept relative to one maximum, relative to another: times 2^by, in two halves, because 2^by alone may be zero where the total is not (maxima hold the values' powers, totals do not).
__device__ __forceinline__ float moved(float total, float by) {
  const float half_of = exp2_approx(0.5f * by);
  return total * half_of * half_of;
}

// Where row r of a head of keys goes.
template <class T>
__device__ __forceinline__ T* out_row(const TreeParams& p, int b, int g, int r) {
  const int t = r / p.group, head = g * p.group + (r - t * p.group);
  return static_cast<T*>(p.a.out) + b * p.a.out_stride[0] + t * p.a.out_stride[1] + head * p.a.out_stride[2];
}
// Stores N values of a row's result; padding, and rows that see nothing, are zero.  `odd`: infinities and NaN of drafted values are added for those that see them.
template <class T, int N>
__device__ __forceinline__ void put_result(const TreeParams& p, int b, int g, int r, unsigned long long mask, int c, float (&v)[N], float sum, bool odd) {
  const bool none = mask == 0 || sum == 0.f;
  const float f = 1.f / (sum * power_of_two(-kTotalPower));
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] *= f;
  if (odd) {
    for (int j = 0; j < p.a.tokens; ++j) {
      if (!(mask >> j & 1)) continue;
      const uint16_t* from = static_cast<const uint16_t*>(p.a.v) + b * p.a.v_stride[0] + j * p.a.v_stride[1] + g * p.a.v_stride[2] + c;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((from[i] & Half16<T>::kExponent) == Half16<T>::kExponent) v[i] += Half16<T>::value(from[i]);
    }
  }
  T* out = out_row<T>(p, b, g, r) + c;
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<uint2*>(out + i) = none ? make_uint2(0u, 0u) : make_uint2(Half16<T>::pack(v[i], v[i + 1]), Half16<T>::pack(v[i + 2], v[i + 3]));
}
// Words of a partial: what is not there yet is zero, so a zero is stored as minus zero.
__device__ __forceinline__ uint32_t word_of(float x) { return __float_as_uint(x) == 0 ? 0x80000000u : __float_as_uint(x); }
__device__ __forceinline__ uint32_t least_of(const uint4& v) { return min(min(v.x, v.y), min(v.z, v.w)); }
__device__ __forceinline__ uint32_t load_word(const float* at) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 load_words(const float* at) {
  uint4 v;
  asm volatile("ld.relaxed.gpu.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ void store_word(float* at, uint32_t v) { asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void store_words(float* at, const uint4& v) {
  asm volatile("st.relaxed.gpu.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Values c .. c + N - 1 of a row, and by one thread its maximum and total, into a partial.
template <int D, int N>
__device__ __forceinline__ void put_partial(float* slot, int r, int c, const float (&v)[N], float most, float sum) {
#pragma unroll
  for (int i = 0; i < N; i += 4) store_words(slot + r * D + c + i, make_uint4(word_of(v[i]), word_of(v[i + 1]), word_of(v[i + 2]), word_of(v[i + 3])));
  if (c == 0) {
    store_word(slot + kRowTile * D + r, word_of(most));
    store_word(slot + kRowTile * (D + 1) + r, word_of(sum));
  }
}
// How an item's partials become one.  Contributors are the CTAs first .. last; their last one adds all up - or, where they are many, the last of every
// `step` adds up a group, and the last of all what the groups have made.  It does so when its own range is done, and waits (with a limit) for CTAs of lower numbers only, which
// were dispatched before it and wait for still lower ones.  A word that has been read is made zero again for the next launch.  No fence and no counter: a fence behind copies
// in flight takes 2.5 us, and a counter that all contributors add to, with one before and one behind it, took 5 us a partial.
//
// Partials whose words are on their way together, and contributors of a group.  Cycles from the end of a range to the end of a join, with 2 / 4 / 6 / 12 together (code that runs once is
// fetched as it runs, and unrolled code is long): two to three contributors 4280 / 4230 / 4480 / 6630, 25 in one step 23600 / 17500 / 16900 / 18500.
// What bounds a join is instructions: a round of two partials of sixteen rows took 2200 cycles when all words were there at the first poll, as long with twice as many words on their way.  With fewer of them
// (no decoding, the least word in place of a chain of tests, one address a partial; this code) 4 tokens, 64 heads over 8, over 8192 / 32768: 33.4 / 45.0 -> 29.7 / 42.0 us, 3 x 1 over 65537: 43.9 -> 42.4.
// Not kept: the next words on their way while some are added up (0 to 3 %); all partials copied into shared memory, and again until they are there (43.5 -> 52).
constexpr int kPartialsTogether = 4;
__device__ __forceinline__ int join_step(int count) {
  if (count <= kPartialsTogether) return count;
  int step = kPartialsTogether;
  while (step * step < count) ++step;
  return step;
}

template <int D>
__device__ __forceinline__ int swizzle(int row) { return D == 128 ? row & 7 : row >> 1 & 3; }      // of 16-byte pieces of rows of D bytes, as TMA's
__device__ __forceinline__ void lds64(uint32_t (&v)[2], uint32_t addr) { asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory"); }
__device__ __forceinline__ void lds128(uint32_t* v, uint32_t addr) { asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory"); }
// a barrier of the warps that compute; whether any of them says so
__device__ __forceinline__ bool any_worker(bool mine) {
  int any;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbar.red.or.pred q, 1, %2, p;\nselp.s32 %0, 1, 0, q;\n}\n" : "=r"(any) : "r"((int)mine), "n"(kWorkers) : "memory");
  return any != 0;
}
__device__ __forceinline__ void workers_sync() { named_bar_sync(1, kWorkers); }

// ldmatrix of what makes two operands
__device__ __forceinline__ void ldsm_two(uint32_t (&a)[2], uint32_t (&b)[2], uint32_t addr) {
  uint32_t r[4];
  ldsm(r, addr);
  a[0] = r[0]; a[1] = r[1]; b[0] = r[2]; b[1] = r[3];
}
__device__ __forceinline__ void ldsm_t_two(uint32_t (&a)[2], uint32_t (&b)[2], uint32_t addr) {
  uint32_t r[4];
  ldsm_t(r, addr);
  a[0] = r[0]; a[1] = r[1]; b[0] = r[2]; b[1] = r[3];
}
// (not volatile: to be moved between the steps of other chains)
__device__ __forceinline__ void mma_halves(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Where the exponents of a token's key and value are in their words (bits), and whether it is seen.
// (A word lies in the same four bytes of memory as its byte, so it can be read where that can.)
constexpr uint32_t kUnseen = 1u << 31;
__device__ __forceinline__ uint32_t where_of(const void* key_power, const void* value_power) {
  return (uint32_t)(reinterpret_cast<uintptr_t>(key_power) & 3) * 8 | (uint32_t)(reinterpret_cast<uintptr_t>(value_power) & 3) * (8 << 8);
}

// Of a thread's two tokens: 2^x scale log2(e); y; from the exponent of a weight to that of what it adds to the total.
struct Constants {
  float key_by[2], value_power[2], to_total[2];
};

template <class T, int D, int NT, int RW>
__global__ void __launch_bounds__(kThreads, Cfg<D, NT, RW>::kCtas) tree_attention_fp8_kernel(const __grid_constant__ Fp8Params params, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D, NT, RW>;
  constexpr int S = C::kStages, kParts = D / 16;                     // 16-byte pieces of a cached row, half of a drafted one's
  constexpr int kSlot = slot_floats<D>();
  constexpr bool kHalf = Half16<T>::kMmaFormat == 0;                 // 16-bit operands are fp16 as they come
  const Fp8Params& p = params;
  const fp6m_tree_attention_args& a = p.a;
  const fp6m_cache_scales& sc = params.scales;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = smem_u32(smem), full = base + C::kBars, empty = full + 8 * S;
  uint32_t* powers = reinterpret_cast<uint32_t*>(smem + C::kPowers);
  uint32_t* where = reinterpret_cast<uint32_t*>(smem + C::kWhere);
  float* pool = reinterpret_cast<float*>(smem + C::kPool);
  float2* stats = reinterpret_cast<float2*>(smem + C::kStats);
  unsigned long long* masks = reinterpret_cast<unsigned long long*>(smem + C::kMasks);
  Plan* plan = reinterpret_cast<Plan*>(smem + C::kPlan);

  const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31, cta = blockIdx.x;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full + 8 * s, 128);                                  // the copying lanes, for what they have stored and for their copies
      mbar_init(empty + 8 * s, 4);                                   // the warps that compute
    }
    mbar_fence_init();
  }
  if (tid == 32 * 4 && p.run > 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 0) make_plan<TilesApart>(p, plan, kLeastUnits, kSlack);
  __syncthreads();
  const long long units = plan->units;
  const int ctas = plan->ctas;
  if (cta >= ctas) return;
  Ranges seg(p, *plan);
  bool dead = false;

  if (warp >= 4) {
    // ==================================================================== copies: a warp the keys and values, one the powers of two
    const bool copies = warp == 4;
    // A granule is p.grain tokens of a page that start at a multiple of their number: those that a TMA copy brings, or fewer.  A warp keeps the pages of 64 granules, two
    // a lane, and those of the next 64 are on their way.  A token's powers of two, a byte each, come as the words that hold them.
    const int grain_log2 = __ffs(p.grain) - 1;
    const int step_slots = kTile % a.page_size;
    bool missing = false;
    int stage = 0;
    uint32_t phase = 1;                                              // of `empty`; the first round of stages is free
#pragma unroll 1
    while (__shfl_sync(0xffffffffu, (int)seg.next(p), 0)) {
      // What decides about the copies is made uniform to the compiler (read from lane 0): TMA copies with operands that differ between lanes take longer to issue.
      const int t0 = __shfl_sync(0xffffffffu, seg.t0, 0), t1 = __shfl_sync(0xffffffffu, seg.t1, 0), length = __shfl_sync(0xffffffffu, seg.length, 0);
      const int g = __shfl_sync(0xffffffffu, seg.item, 0), tiles = __shfl_sync(0xffffffffu, seg.tiles, 0);
      const int* table = a.page_table + seg.b * a.page_table_stride;
      const uint8_t *k_powers = static_cast<const uint8_t*>(sc.k_scales) + g * sc.k_scales_stride[2], *v_powers = static_cast<const uint8_t*>(sc.v_scales) + g * sc.v_scales_stride[2];
      int pages[2], next_pages[2], slot[2];
      auto look_up = [&](int block, int (&into)[2]) {                // the pages of granules 64 block ..
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const long long j = ((long long)block * 64 + 32 * i + lane) << grain_log2;
          into[i] = j < length ? table[(int)((unsigned long long)j * p.page_magic >> p.page_shift)] : -1;
        }
      };
      look_up(t0 >> grain_log2, pages);
      look_up((t0 >> grain_log2) + 1, next_pages);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = t0 * kTile + 32 * i + lane;
        slot[i] = j - (int)((unsigned long long)j * p.page_magic >> p.page_shift) * a.page_size;
      }
#pragma unroll 1
      for (int tile = t0; tile < t1; ++tile) {
        const int at_block = tile & (p.grain - 1);                   // tiles of a block: as many as tokens of a granule
        if (at_block == 0 && tile != t0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) pages[i] = next_pages[i];
          look_up((tile >> grain_log2) + 1, next_pages);
        }
        const bool drafted = tile + 1 == tiles, by_tma = p.run > 0 && (tile + 1) * kTile <= length;
        const uint32_t keys = base + stage * C::kStageBytes, values = keys + C::kTileBytes, bar = full + 8 * stage;
        auto page_at = [&](int granule) {                            // of the tile
          const int in = (at_block << (6 - grain_log2)) + granule, lo = __shfl_sync(0xffffffffu, pages[0], in & 31), hi = __shfl_sync(0xffffffffu, pages[1], in & 31);
          return in < 32 ? lo : hi;
        };
        mbar_wait_bounded<20>(empty + 8 * stage, phase, p.status, dead);
        if (copies && by_tma) {
          if (elect_one()) mbar_expect_tx(bar, C::kStageBytes);
          __syncwarp();
          const int first_slot = __shfl_sync(0xffffffffu, slot[0], 0);
          auto bring = [&](auto runs) {
            constexpr int R = decltype(runs)::value;
            int page[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const int of = page_at(r);
              page[r] = (unsigned)of < (unsigned)a.pages ? of : a.pages;       // behind the last page the copy reads zeros
            }
            if (elect_one()) {
              int at = first_slot;
#pragma unroll
              for (int r = 0; r < R; ++r) {
                tma_load_run(keys + r * (kTile / R) * D, &kmap, 0, g, at, page[r], bar);
                tma_load_run(values + r * (kTile / R) * D, &vmap, 0, g, at, page[r], bar);
                at += kTile / R;
                if (at == a.page_size) at = 0;
              }
            }
            __syncwarp();
          };
          if (p.run == 64) bring(std::integral_constant<int, 1>());
          else if (p.run == 32) bring(std::integral_constant<int, 2>());
          else if (p.run == 16) bring(std::integral_constant<int, 4>());
          else bring(std::integral_constant<int, 8>());
        } else if (copies && drafted) {
          constexpr int kWide = D / 8;
          const int part = lane % kWide;
          for (int row = lane / kWide; row < a.tokens; row += 32 / kWide) {
            const uint32_t to = row * 2 * D + ((part ^ (row & 7)) * 16);
            copy16(keys + to, static_cast<const T*>(a.k) + seg.b * a.k_stride[0] + row * a.k_stride[1] + g * a.k_stride[2] + part * 8, 16);
            copy16(values + to, static_cast<const T*>(a.v) + seg.b * a.v_stride[0] + row * a.v_stride[1] + g * a.v_stride[2] + part * 8, 16);
          }
        } else if (!drafted) {
          int page[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            page[i] = page_at((32 * i + lane) >> grain_log2);
            const bool there = tile * kTile + 32 * i + lane < length;
            missing = missing || (there && (unsigned)page[i] >= (unsigned)a.pages);
            if (!there || (unsigned)page[i] >= (unsigned)a.pages) page[i] = -1;
          }
          if (!copies) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t at_word = kUnseen;                              // any score becomes minus infinity, a weight of zero
              if (page[i] >= 0) {
                auto in = [&](const long long (&stride)[3]) { return (unsigned long long)(unsigned)page[i] * (unsigned)stride[0] + (unsigned long long)(unsigned)slot[i] * (unsigned)stride[1]; };
                const uint8_t *k = k_powers + in(sc.k_scales_stride), *v = v_powers + in(sc.v_scales_stride);
                const uint32_t to = base + C::kPowers + (stage * 2 * kTile + 32 * i + lane) * 4;
                copy4(to, reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(k) & ~(uintptr_t)3));
                copy4(to + kTile * 4, reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(v) & ~(uintptr_t)3));
                at_word = where_of(k, v);
              }
              where[stage * kTile + 32 * i + lane] = at_word;
            }
          } else {
            const uint8_t *k[2], *v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              k[i] = page[i] >= 0 ? static_cast<const uint8_t*>(a.k_cache) + page[i] * a.k_cache_stride[0] + slot[i] * a.k_cache_stride[1] + g * a.k_cache_stride[2] : nullptr;
              v[i] = page[i] >= 0 ? static_cast<const uint8_t*>(a.v_cache) + page[i] * a.v_cache_stride[0] + slot[i] * a.v_cache_stride[1] + g * a.v_cache_stride[2] : nullptr;
            }
            const int part = lane % kParts;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll 4
              for (int r0 = 0; r0 < 32; r0 += 32 / kParts) {
                const int in = r0 + lane / kParts, row = 32 * i + in;
                const uint8_t* from_k = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k[i]), in));
                const uint8_t* from_v = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v[i]), in));
                const uint32_t to = row * D + ((part ^ swizzle<D>(row)) * 16);
                copy16(keys + to, from_k ? from_k + part * 16 : static_cast<const uint8_t*>(a.q), from_k ? 16 : 0);
                copy16(values + to, from_v ? from_v + part * 16 : static_cast<const uint8_t*>(a.q), from_v ? 16 : 0);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          slot[i] += step_slots;
          if (slot[i] >= a.page_size) slot[i] -= a.page_size;
        }
        // (the arrival of asynchronous copies does not order a thread's stores, a plain one does)
        copies_arrive(bar);
        mbar_arrive(bar);
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
    }
    if (missing && p.status) atomicExch(p.status, FP6M_ERR_BAD_ARG);
    return;
  }

  // ====================================================================== scores, weights, sums: a warp has sixteen tokens of a tile and all rows
  const int quad = lane >> 2, col = lane & 3;                        // tokens quad and quad + 8; of eight rows 2 col and 2 col + 1; values 2 quad and 2 quad + 1 of sixteen
  const int row_warp = warp / C::kKeyWarps, key_warp = warp % C::kKeyWarps, group0 = row_warp * NT;      // this warp's share of the rows and of the tokens, its first group of rows
  int stage = 0;
  uint32_t phase = 0;
  bool joins = false, join_odd = false;                              // the item of this CTA's first segment, if it started before
  int join_b = 0, join_g = 0, join_first = 0, join_last = 0;
#pragma unroll 1
  while (seg.next(p)) {
    const int g = seg.item, rows = p.rows;
    // ---- queries: fp16, and for bf16 the power of two of each row
    uint32_t q[C::kSharedQueries ? 1 : kParts][2];
    float row_by[NT][2];
    uint2* shared_q = reinterpret_cast<uint2*>(smem + C::kQueries);
    float* shared_row_by = reinterpret_cast<float*>(smem + C::kQueries + kParts * C::kGroups * 32 * 8);
    auto load_queries = [&](int n, auto&& put) {                     // of rows 8 n .. 8 n + 7: this thread's values of row 8 n + quad
      const int r = 8 * n + quad;
      const T* src = nullptr;
      if (r < rows) {
        const int t = r / p.group, head = g * p.group + (r - t * p.group);
        src = static_cast<const T*>(a.q) + seg.b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2];
      }
      uint2 four[kParts];
#pragma unroll
      for (int i = 0; i < kParts; ++i) four[i] = src ? *reinterpret_cast<const uint2*>(src + 16 * i + 4 * col) : make_uint2(0u, 0u);
      int x = 0;
      if constexpr (!kHalf) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < kParts; ++i) most = fmaxf(most, fmaxf(largest_of<T>(four[i].x), largest_of<T>(four[i].y)));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        x = exponent_for_half(most);
        const float down = power_of_two(-x);
#pragma unroll
        for (int i = 0; i < kParts; ++i) four[i] = make_uint2(scaled_halves<T>(four[i].x, down), scaled_halves<T>(four[i].y, down));
      }
#pragma unroll
      for (int i = 0; i < kParts; ++i) put(i, four[i]);
      return power_of_two(x);
    };
    if constexpr (C::kSharedQueries) {
      if (warp < C::kGroups) {
        const float by = load_queries(warp, [&](int i, uint2 four) { shared_q[(i * C::kGroups + warp) * 32 + lane] = four; });
        if (col == 0) shared_row_by[8 * warp + quad] = by;
      }
      workers_sync();
      if constexpr (!kHalf) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) row_by[n][e] = shared_row_by[8 * (group0 + n) + 2 * col + e];
      }
    } else {
      const float by = load_queries(0, [&](int i, uint2 four) {
        q[i][0] = four.x;
        q[i][1] = four.y;
      });
      if constexpr (!kHalf) {
#pragma unroll
        for (int e = 0; e < 2; ++e) row_by[0][e] = __shfl_sync(0xffffffffu, by, (2 * col + e) * 4);
      }
    }
    float o[kParts][NT][4], top[NT][2], total[NT][2];                // sums: even value of two rows, odd value of two rows
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < kParts; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
      top[n][0] = top[n][1] = -INFINITY;
      total[n][0] = total[n][1] = 0.f;
    }
    bool odd = false;                                                // infinities or NaN among the drafted values
    // M tiles' scores of sixteen tokens each -> weights for the second product (fp16), with the running maximum and sum
    auto weigh = [&](auto tiles, float (&s)[decltype(tiles)::value][NT][4], const Constants (&of)[decltype(tiles)::value], bool drafted, uint32_t (&w)[decltype(tiles)::value][NT][2]) {
      constexpr int M = decltype(tiles)::value;
      bool grows = false;
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[m][n][e] = fmaf(s[m][n][e], kHalf ? of[m].key_by[e >> 1] : of[m].key_by[e >> 1] * row_by[n][e & 1], of[m].value_power[e >> 1]);
            if (drafted) {
              const int t = key_warp * 16 + quad + (e & 2) * 4;
              if (t >= a.tokens || !(masks[8 * (group0 + n) + 2 * col + (e & 1)] >> t & 1)) s[m][n][e] = -INFINITY;
            }
            grows = grows || s[m][n][e] > top[n][e & 1] + kGrowth;
          }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float now = top[n][e];
#pragma unroll
            for (int m = 0; m < M; ++m) now = fmaxf(now, fmaxf(s[m][n][e], s[m][n][2 + e]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
            const float by = top[n][e] - (now == -INFINITY ? 0.f : now);
            keep[e] = exp2_approx(by);
            top[n][e] = now;
            total[n][e] = moved(total[n][e], by);
          }
#pragma unroll
          for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][n][e] *= keep[e & 1];
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float below[2] = {top[n][0] == -INFINITY ? 0.f : top[n][0], top[n][1] == -INFINITY ? 0.f : top[n][1]};
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[m][n][e] - below[e & 1];
            s[m][n][e] = exp2_approx(x);
            total[n][e & 1] += exp2_approx(x + of[m].to_total[e >> 1]);
          }
          w[m][n][0] = transposed(Half16<half>::pack(s[m][n][0], s[m][n][1]));
          w[m][n][1] = transposed(Half16<half>::pack(s[m][n][2], s[m][n][3]));
        }
      }
    };
    auto queries_of = [&](int i, uint32_t (&b)[NT][2]) {              // of sixteen values, all groups
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (C::kSharedQueries) {
          const uint2 two = shared_q[(i * C::kGroups + group0 + n) * 32 + lane];
          b[n][0] = two.x;
          b[n][1] = two.y;
        } else {
          b[n][0] = q[i][0];
          b[n][1] = q[i][1];
        }
      }
    };
    // Sixteen cached tokens of each of M tiles, or M times sixteen of one, from the stage on that is next; side by side, so that one chain of latencies serves all.
    auto cached_tiles = [&](auto parts) {
      constexpr int M = decltype(parts)::value;
      int at[M], first[M];
      at[0] = stage;
      first[0] = key_warp * (RW == 1 ? 16 : 32);
      if constexpr (M == 2) {
        at[1] = RW == 2 ? stage : stage + 1 == S ? 0 : stage + 1;
        first[1] = first[0] + (RW == 1 ? 0 : 16);
      }
      float s[M][NT][4] = {};
      Constants of[M];
      uint32_t w[M][NT][2];
      const int in = lane & 15;
#pragma unroll
      for (int m = 0; m < M; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = first[m] + quad + 8 * e;
          const uint32_t place = where[at[m] * kTile + j], kw = powers[at[m] * 2 * kTile + j], vw = powers[(at[m] * 2 + 1) * kTile + j];
          const int x = (int)(kw >> (place & 31) & 255) - 127, y = (int)(vw >> (place >> 8 & 31) & 255) - 127;
          of[m].key_by[e] = place == kUnseen ? 0.f : power_of_two(x) * p.scale_log2;
          of[m].value_power[e] = place == kUnseen ? -INFINITY : (float)y;
          of[m].to_total[e] = (float)(kTotalPower - y);
        }
      }
#pragma unroll
      for (int i = 0; i < kParts; i += 2) {
        uint32_t k[M][2][2];
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const int row = first[m] + in;
          ldsm_two(k[m][0], k[m][1], base + at[m] * C::kStageBytes + row * D + (((i + (lane >> 4)) ^ swizzle<D>(row)) * 16));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t b[NT][2];
          queries_of(i + c, b);
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const uint32_t operand[4] = {halves_of(k[m][c][0]), halves_of(k[m][c][1]), upper_halves_of(k[m][c][0]), upper_halves_of(k[m][c][1])};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_halves(s[m][n], operand, b[n][0], b[n][1]);
          }
        }
      }
      weigh(parts, s, of, false, w);
#pragma unroll
      for (int i = 0; i < kParts; i += 2) {
        uint32_t v[M][2][2];
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const int row = first[m] + in;
          ldsm_t_two(v[m][0], v[m][1], base + at[m] * C::kStageBytes + C::kTileBytes + row * D + (((i + (lane >> 4)) ^ swizzle<D>(row)) * 16));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            // two tokens' values 2 n and 2 n + 1 -> the two tokens' values 2 n, then those 2 n + 1
            const uint32_t x = prmt(v[m][c][0], 0, 0x3120), y = prmt(v[m][c][1], 0, 0x3120);
            const uint32_t operand[4] = {halves_of(x), upper_halves_of(x), halves_of(y), upper_halves_of(y)};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_halves(o[i + c][n], operand, w[m][n][0], w[m][n][1]);
          }
      }
    };
    // The drafted tokens: fp16 with a power of two each; of the values the even ones of 16 before the odd ones, which is how E4M3 values come apart above.
    // Infinities and NaN of values must not meet a weight of zero: they are zero here, and added to the rows that see them at the end.
    auto drafted_tile = [&] {
      const uint32_t keys = base + stage * C::kStageBytes, values = keys + C::kTileBytes;
      const int padded = (a.tokens + 15) & ~15;
      bool mine_odd = false;
      if (tid < 8 * C::kGroups) masks[tid] = tid < rows ? mask_of(p, seg.b, tid / p.group) : 0;
#pragma unroll 1
      for (int i0 = 0; i0 < 2 * padded * kParts; i0 += kWorkers) {
        const int i = i0 + tid, row = i / kParts % padded, part = i % kParts;
        const bool is_value = i / kParts >= padded, lives = i < 2 * padded * kParts, there = lives && row < a.tokens;
        const uint32_t at = (is_value ? values : keys) + row * 2 * D;
        const uint32_t lo = at + (((2 * part) ^ (row & 7)) * 16), hi = at + (((2 * part + 1) ^ (row & 7)) * 16);
        uint32_t w[8] = {};
        if (there) {
          lds128(w, lo);
          lds128(w + 4, hi);
        }
        if (is_value) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            constexpr uint32_t E = Half16<T>::kExponent;
            if ((w[e] & E) == E) { w[e] &= 0xffff0000u; mine_odd = true; }
            if ((w[e] >> 16 & E) == E) { w[e] &= 0xffffu; mine_odd = true; }
          }
        }
        int x = 0;
        if constexpr (!kHalf) {
          float most = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, largest_of<T>(w[e]));
#pragma unroll
          for (int d = 1; d < kParts; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
          x = exponent_for_half(most);
          if (is_value) x = max(x, kLeastPower);
          const float down = power_of_two(-x);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = scaled_halves<T>(w[e], down);
        }
        if (lives) {
          if (is_value) {
            const uint32_t even[4] = {prmt(w[0], w[1], 0x5410), prmt(w[2], w[3], 0x5410), prmt(w[4], w[5], 0x5410), prmt(w[6], w[7], 0x5410)};
            const uint32_t uneven[4] = {prmt(w[0], w[1], 0x7632), prmt(w[2], w[3], 0x7632), prmt(w[4], w[5], 0x7632), prmt(w[6], w[7], 0x7632)};
#pragma unroll
            for (int e = 0; e < 4; ++e) { w[e] = even[e]; w[4 + e] = uneven[e]; }
          }
          if (part == 0) powers[(stage * 2 + is_value) * kTile + row] = (uint32_t)x;
          sts128(lo, w);
          sts128(hi, w + 4);
        }
      }
      odd = any_worker(mine_odd);
      const int first = key_warp * 16;
      if (first >= padded) return;
      float s[1][NT][4] = {};
      Constants of[1];
      uint32_t w[1][NT][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = (int)powers[stage * 2 * kTile + first + quad + 8 * e], y = (int)powers[(stage * 2 + 1) * kTile + first + quad + 8 * e];
        of[0].key_by[e] = power_of_two(x) * p.scale_log2;
        of[0].value_power[e] = (float)y;
        of[0].to_total[e] = (float)(kTotalPower - y);
      }
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        uint32_t k0[2], k1[2];                                       // (rows that are eight apart are swizzled alike)
        const uint32_t at = keys + (first + quad) * 2 * D + (((2 * i + (col >> 1)) ^ (quad & 7)) * 16) + (col & 1) * 8;
        lds64(k0, at);
        lds64(k1, at + 8 * 2 * D);
        const uint32_t operand[4] = {k0[0], k1[0], k0[1], k1[1]};
        uint32_t b[NT][2];
        queries_of(i, b);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_halves(s[0][n], operand, b[n][0], b[n][1]);
      }
      weigh(std::integral_constant<int, 1>(), s, of, true, w);
      const int row = first + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        uint32_t wide[4];
        ldsm_t(wide, values + row * 2 * D + (((2 * i + (lane >> 3 & 1)) ^ (row & 7)) * 16));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_halves(o[i][n], wide, w[0][n][0], w[0][n][1]);
      }
    };
    // waits for the stage that is next, and gives it back
    auto take = [&](int at) { mbar_wait_bounded<20>(full + 8 * at, at < stage ? phase ^ 1 : phase, p.status, dead); };
    auto give_back = [&](bool other_copies) {
      if (other_copies) fence_async_proxy();                         // (what TMA did not bring is overwritten by it perhaps)
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * stage);
      if (++stage == S) { stage = 0; phase ^= 1; }
    };
#pragma unroll 1
    for (int tile = seg.t0; tile < seg.t1;) {
      const bool other_copies = p.run == 0 || (tile + C::kTogether) * kTile > seg.length;
      take(stage);
      if (C::kTogether == 2 && tile + 1 < min(seg.t1, seg.tiles - 1)) {
        take(stage + 1 == S ? 0 : stage + 1);
        cached_tiles(std::integral_constant<int, 2>());
        give_back(other_copies);
        give_back(other_copies);
        tile += 2;
      } else {
        if (tile + 1 == seg.tiles) drafted_tile();
        else cached_tiles(std::integral_constant<int, RW>());
        give_back(other_copies);
        ++tile;
      }
    }

    // ---- the end of this CTA's keys for these rows: the warps pool their sums
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) total[n][e] += __shfl_xor_sync(0xffffffffu, total[n][e], d);
        if (quad == 0) stats[warp * 8 * NT + 8 * n + 2 * col + e] = make_float2(top[n][e], total[n][e]);
      }
    const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
    float* slot = p.partials + (size_t)(kSlots * cta + (seg.t0 == 0 ? 1 : 0)) * kSlot;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (8 * n >= rows) break;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (8 * (group0 + n) + 2 * col + e < rows) {
          float* to = pool + (warp * 8 + 2 * col + e) * C::kPoolRow + 2 * quad;
#pragma unroll
          for (int i = 0; i < kParts; ++i) *reinterpret_cast<float2*>(to + 16 * i) = make_float2(o[i][n][e], o[i][n][2 + e]);
        }
      workers_sync();
      constexpr int V = D / 16;                                      // values of a thread
      const int in = tid >> 4, c = (tid & 15) * V;
#pragma unroll
      for (int rw = 0; rw < RW; ++rw) {
        const int r = 8 * (rw * NT + n) + in;
        if (r >= rows) break;
        float2 of[C::kKeyWarps];
        float most = -INFINITY, sum = 0.f, v[V] = {};
#pragma unroll
        for (int k = 0; k < C::kKeyWarps; ++k) {
          of[k] = stats[(rw * C::kKeyWarps + k) * 8 * NT + 8 * n + in];
          most = fmaxf(most, of[k].x);
        }
#pragma unroll
        for (int k = 0; k < C::kKeyWarps; ++k) {
          const float by = of[k].x - (most == -INFINITY ? 0.f : most), f = exp2_approx(by);
          sum += moved(of[k].y, by);
          const float4* from = reinterpret_cast<const float4*>(pool + ((rw * C::kKeyWarps + k) * 8 + in) * C::kPoolRow + c);
#pragma unroll
          for (int i = 0; i < V / 4; ++i) {
            const float4 x = from[i];
            v[4 * i] = fmaf(x.x, f, v[4 * i]);
            v[4 * i + 1] = fmaf(x.y, f, v[4 * i + 1]);
            v[4 * i + 2] = fmaf(x.z, f, v[4 * i + 2]);
            v[4 * i + 3] = fmaf(x.w, f, v[4 * i + 3]);
          }
        }
        if (whole) put_result<T>(p, seg.b, g, r, masks[r], c, v, sum, odd);
        else put_partial<D>(slot, r, c, v, most, sum);
      }
      workers_sync();
    }
    if (seg.t0 == 0) continue;
    joins = true;
    join_odd = odd;
    join_b = seg.b;
    join_g = g;
    join_first = cta_of(units, ctas, seg.unit + p.overhead);
    join_last = cta_of(units, ctas, seg.unit + p.overhead + seg.tiles - 1);
  }

  if (!joins) return;
  const int count = join_last - join_first + 1, step = join_step(count), group = (cta - join_first) / step;
  const bool ends = cta == join_last;
  if (!ends && (cta - join_first) % step != step - 1) return;
  // the sums of the groups before (if this is the last CTA), then the partials of this group
  const int before = ends ? group : 0, members = cta - join_first - group * step + 1;
  auto source = [&](int k) {                                         // (offsets fit an int)
    const int c = join_first + group * step + k - before;
    return p.partials + (k < before ? (kSlots * (join_first + k * step + step - 1) + 2) * kSlot : (kSlots * c + (c == join_first ? 1 : 0)) * kSlot);
  };
  // Few instructions a word: one warp per scheduler goes through this, with nothing beside it.  A thread has four values, and 64 behind them four more (D = 128), of a row, or of two that are
  // eight apart.
  constexpr int V = D / 16, R = C::kGroups > 1 ? 2 : 1, K = kPartialsTogether / R;
  const int c = (tid & 15) * 4, total_sources = before + members;
#pragma unroll 1
  for (int r0 = tid >> 4; r0 < p.rows; r0 += 8 * R) {
    float most[R], sum[R] = {}, v[R][V] = {};
    const bool second = R == 2 && r0 + 8 < p.rows;
#pragma unroll
    for (int i = 0; i < R; ++i) most[i] = -INFINITY;
    const int at_values = r0 * D + c, at_stats = kRowTile * D + r0, next_values = second ? 8 * D : 0, next_stats = second ? 8 : 0;
#pragma unroll 1
    for (int k0 = 0; k0 < total_sources; k0 += K) {
      float* from[K];
      uint4 x[R][K][V / 4];
      uint32_t m[R][K], t[R][K];
#pragma unroll
      for (int e = 0; e < K; ++e) from[e] = source(min(k0 + e, total_sources - 1));
      bool there = false;
      for (uint32_t polls = 0; !there; ++polls) {
        uint32_t least = ~0u;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < K; ++e) {
            const float *stats_at = from[e] + at_stats + (i ? next_stats : 0), *values_at = from[e] + at_values + (i ? next_values : 0);
            m[i][e] = load_word(stats_at);
            t[i][e] = load_word(stats_at + kRowTile);
#pragma unroll
            for (int j = 0; j < V / 4; ++j) x[i][e][j] = load_words(values_at + 64 * j);
          }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < K; ++e) {
            least = min(least, min(m[i][e], t[i][e]));
#pragma unroll
            for (int j = 0; j < V / 4; ++j) least = min(least, least_of(x[i][e][j]));
          }
        there = least != 0;
        if (dead || polls > 1u << 19) {                              // (a round takes about a microsecond)
          if (!dead && p.status) atomicExch(p.status, FP6M_ERR_TIMEOUT);
          dead = there = true;
        }
      }
      // the sixteen threads of a row are neighbours in a warp, and have all read it now
      __syncwarp(0xffffu << (lane & 16));
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float now = most[i];
#pragma unroll
        for (int e = 0; e < K; ++e) now = fmaxf(now, __uint_as_float(m[i][e]));
        const float below = now == -INFINITY ? 0.f : now, keep = exp2_approx(most[i] - below);
        sum[i] = moved(sum[i], most[i] - below);
        most[i] = now;
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] *= keep;
#pragma unroll
        for (int e = 0; e < K; ++e) {
          const bool counts = k0 + e < total_sources;
          const float by = counts ? __uint_as_float(m[i][e]) - below : -INFINITY, f = exp2_approx(by);
          sum[i] += moved(__uint_as_float(t[i][e]), by);
#pragma unroll
          for (int j = 0; j < V / 4; ++j) {
            v[i][4 * j] = fmaf(__uint_as_float(x[i][e][j].x), f, v[i][4 * j]);
            v[i][4 * j + 1] = fmaf(__uint_as_float(x[i][e][j].y), f, v[i][4 * j + 1]);
            v[i][4 * j + 2] = fmaf(__uint_as_float(x[i][e][j].z), f, v[i][4 * j + 2]);
            v[i][4 * j + 3] = fmaf(__uint_as_float(x[i][e][j].w), f, v[i][4 * j + 3]);
          }
          if (counts && (i == 0 || second)) {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) store_words(from[e] + at_values + 8 * D * i + 64 * j, make_uint4(0, 0, 0, 0));
            if (c == 0) {
              store_word(from[e] + at_stats + 8 * i, 0);
              store_word(from[e] + at_stats + kRowTile + 8 * i, 0);
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i && !second) continue;
      const int r = r0 + 8 * i;
      const unsigned long long mask = ends ? mask_of(p, join_b, r / p.group) : 0;
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        float four[4] = {v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3]};
        if (ends) put_result<T>(p, join_b, join_g, r, mask, c + 64 * j, four, sum[i], join_odd);
        else put_partial<D>(p.partials + (size_t)(kSlots * cta + 2) * kSlot, r, c + 64 * j, four, most[i], sum[i]);
      }
    }
  }
}

int fp8_ctas(int sms, int per_sm) {
  const int want = sms > 0 ? per_sm * sms : kMaxTreeCtas;
  return want < kMaxTreeCtas ? want : kMaxTreeCtas;
}

template <class T, int D, int NT, int RW>
cudaError_t launch_groups(const Fp8Params& p, int sms, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
  using C = Cfg<D, NT, RW>;
  cudaError_t e = allow_shared_memory<tree_attention_fp8_kernel<T, D, NT, RW>>(C::kBytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(tree_attention_fp8_kernel<T, D, NT, RW>, dim3(fp8_ctas(sms, C::kCtas)), dim3(kThreads), C::kBytes, stream, p, kmap, vmap);
}
template <class T, int D>
cudaError_t launch_head(const Fp8Params& p, int sms, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
  return p.rows <= 8 ? launch_groups<T, D, 1, 1>(p, sms, kmap, vmap, stream) : p.rows <= 16 ? launch_groups<T, D, 2, 1>(p, sms, kmap, vmap, stream) : launch_groups<T, D, 2, 2>(p, sms, kmap, vmap, stream);
}
cudaError_t launch_fp8(Fp8Params p, int sms, cudaStream_t stream) {
  const fp6m_tree_attention_args& a = p.a;
  p.grain = kTile;
  while (a.page_size % p.grain) p.grain /= 2;
  // swizzled rows come in eights
  p.run = p.grain >= 8 ? p.grain : 0;
  CUtensorMap kmap = {}, vmap = {};
  if (p.run == 0 || a.max_pages == 0 || encode_cache_map(a.k_cache, 1, a.head_dim, a.kv_heads, a.page_size, a.pages, a.k_cache_stride, p.run, &kmap) != cudaSuccess ||
      encode_cache_map(a.v_cache, 1, a.head_dim, a.kv_heads, a.page_size, a.pages, a.v_cache_stride, p.run, &vmap) != cudaSuccess)
    p.run = 0;
  if (a.type == FP6M_TYPE_F16) return a.head_dim == 64 ? launch_head<half, 64>(p, sms, kmap, vmap, stream) : launch_head<half, 128>(p, sms, kmap, vmap, stream);
  return a.head_dim == 64 ? launch_head<__nv_bfloat16, 64>(p, sms, kmap, vmap, stream) : launch_head<__nv_bfloat16, 128>(p, sms, kmap, vmap, stream);
}

size_t few_rows_bytes(int sms) { return (size_t)fp8_ctas(sms, Cfg<128, 1, 1>::kCtas) * kSlots * slot_floats<128>() * sizeof(float); }

}  // namespace

extern "C" {

// (the two kernels keep apart what they leave there)
size_t fp6m_tree_attention_fp8_scratch_bytes(int sms) { return few_rows_bytes(sms) + kCounterBytes + tree_tc5_partial_bytes(sms); }

int fp6m_tree_attention_fp8(const fp6m_tree_attention_args* args, const fp6m_cache_scales* scales, void* scratch, size_t scratch_bytes, int dev, void* stream, int* status_dev) {
  if (!args || !scales) return FP6M_ERR_BAD_ARG;
  const int rc = check_tree_args(*args, 16, scratch);
  if (rc != FP6M_OK || args->batch == 0 || args->tokens == 0 || args->heads == 0) return rc;
  if (args->max_pages > 0 && (!scales->k_scales || !scales->v_scales)) return FP6M_ERR_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (scales->k_scales_stride[i] < 0 || scales->v_scales_stride[i] < 0) return FP6M_ERR_BAD_ARG;
  for (int i = 0; i < 2; ++i)
    if (scales->k_scales_stride[i] > 0xffffffffll || scales->v_scales_stride[i] > 0xffffffffll) return FP6M_ERR_PROB_SHAPE;
  DeviceGuard guard(dev);
  const int sms = sm_count(dev);
  if (sms <= 0) return cuda_fail(cudaGetLastError(), "cudaDeviceGetAttribute");
  if (scratch_bytes < fp6m_tree_attention_fp8_scratch_bytes(sms)) return FP6M_ERR_SCRATCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (args->tokens * (args->heads / args->kv_heads) > kFewRows) {
    e = launch_tree_tc5(tree_params(*args, static_cast<unsigned char*>(scratch) + few_rows_bytes(sms), kCounterBytes, status_dev), scales, sms, st);
  } else {
    Fp8Params p;
    static_cast<TreeParams&>(p) = tree_params(*args, scratch, 0, status_dev);
    p.scales = *scales;
    e = launch_fp8(p, sms, st);
  }
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "tree_attention_fp8 launch");
}

}  // extern "C"
