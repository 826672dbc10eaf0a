// Attention of drafted tokens over a paged cache in 8 bits: as tree_attention.cu, but committed keys and values are E4M3 with a power of two for each
// token and head (cache_fp8.cu writes them).
//
//   k_j = 2^x_j * K_j,  v_j = 2^y_j * V_j     K_j, V_j in E4M3, exact in fp16
//   a_ij = scale * log2(e) * 2^x_j * (q_i . K_j) + y_j,   M_i = max_j a_ij,   w_ij = 2^(a_ij - M_i)
//   o_i  = sum_j w_ij V_j / sum_j 2^-y_j w_ij
//
// so that the scales cost one fused multiply-add per score and none per key or value: the values' power is an addend of the exponent, and the maximum that
// keeps the exponentials in range is that of the weights as they meet the values.  These are rounded once, to fp16 (2^-11 of a weight; below 2^-14 of the largest they
// become multiples of 2^-24), for both types of queries; the sum that they are divided by has them unrounded.  Queries in bf16 come as fp16 times a power of
// two for each row, with the largest value between 2^14 and 2^15: exact but for values 2^-28 times smaller than that.
//
// Drafted keys and values are 16 bits.  They make a tile of their own behind the cached ones, which is brought into the form of the others when it is worked
// on: fp16 with a power of two per token (bf16 as the queries, fp16 as it is).
//
// Work is cut into equal ranges of (sequence, head of keys, row tile, key tile) units as in tree_attention.cu; tiles have 128 cached tokens, as many bytes as 64 there.
#include "device_utils.cuh"
#include "host_common.h"
#include "tree_attention.cuh"

namespace {

using namespace fp6m;

constexpr int kThreads = 128;
constexpr int kTile = 128, kDrafted = 64;          // cached tokens of a tile; places for drafted ones in theirs
constexpr int kStages = 3;
constexpr int kMaxCtas = 512;
constexpr int kLeastUnits = 3, kSlack = 8;
constexpr int kCounterBytes = kMaxCtas * 2 * 3 * 4;
constexpr int kPoolFloats = 3 * 16 * 32;           // what the warps that share keys pool at a time

struct Fp8Params {
  TreeParams tree;
  fp6m_cache_scales scales;
};

// Tiles of cached tokens, then one of the drafted tokens.
struct TilesApart {
  static __device__ __forceinline__ int of(const TreeParams&, int length) { return (length + kTile - 1) / kTile + 1; }
};
using Ranges = SegmentsOf<TilesApart>;

// two E4M3 values in fp16 (exact)
__device__ __forceinline__ uint32_t halves_of(uint32_t two) {
  uint32_t h;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(h) : "r"(two));
  return h;
}
// 2^n, -127 <= n <= 128
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float(n > -127 ? (uint32_t)(n + 127) << 23 : 0x00400000u); }
// the exponent that brings values of up to `top` below 2^15: fp16 holds them and what is up to 2^29 times smaller
__device__ __forceinline__ int exponent_for_half(float top) { return top == 0.f ? 0 : max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100); }
__device__ __forceinline__ float finite_magnitude(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

template <int D>
__device__ __forceinline__ int swizzle(int row) { return D == 128 ? row & 7 : row >> 1 & 3; }      // of 16-byte pieces of rows of D bytes

// kRowTile rows, a warp for every 16 of them; the warps that this leaves share the keys of a tile and pool their sums.
template <class T, int D, int kRowTile>
__global__ void __launch_bounds__(kThreads, 2) tree_attention_fp8_kernel(const __grid_constant__ Fp8Params params) {
  constexpr int kRowWarps = kRowTile / 16, kKeyWarps = 4 / kRowWarps;
  constexpr int kMine = kTile / kKeyWarps, kMyDrafted = kDrafted / kKeyWarps;     // tokens of a tile that a warp works on
  constexpr int kTileBytes = kTile * D, kStageBytes = 2 * kTileBytes;             // keys or values of a tile
  constexpr int kChunks = D / 16, kRowsPerPass = kThreads / kChunks;              // 16-byte pieces of a cached row
  constexpr int kWide = D / 8;                                                    // and of a drafted one
  constexpr int kSlot = slot_floats<D, kRowTile, true>();
  constexpr bool kHalf = sizeof(T) == 2 && Half16<T>::kMmaFormat == 0;            // 16-bit operands are fp16 as they come
  const TreeParams& p = params.tree;
  const fp6m_tree_attention_args& a = p.a;
  const fp6m_cache_scales& sc = params.scales;
  extern __shared__ __align__(128) uint8_t smem[];
  // constants of a tile's tokens: 2^x scale log2(e); y and 2^-y
  float* key_by = reinterpret_cast<float*>(smem + kStages * kStageBytes);                            // [stage][kTile]
  float2* value_by = reinterpret_cast<float2*>(key_by + kStages * kTile);
  float* pool = reinterpret_cast<float*>(value_by + kStages * kTile);
  float* stats = pool + kPoolFloats;                                                // [warp][2][16]: maxima, totals
  const uint8_t** places = reinterpret_cast<const uint8_t**>(stats + 4 * 32);      // [2][keys, values][kTile]: where the tokens of a tile are
  Plan* plan = reinterpret_cast<Plan*>(places + 4 * kTile);
  int* flags = reinterpret_cast<int*>(plan + 1);                                   // [0] a page did not exist, [1] last to arrive

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row_warp = warp / kKeyWarps, key_warp = warp % kKeyWarps;
  if (tid == 0) flags[0] = 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cta = blockIdx.x;
  if (warp == 0) make_plan<TilesApart>(p, plan, kLeastUnits, kSlack);
  __syncthreads();
  const long long units = plan->units;
  const int ctas = plan->ctas;
  if (cta >= ctas) return;
  Ranges seg(p, *plan);

  // ---- copies of a tile, a row of keys and one of values per token.  A thread works out where one token's rows are; the others take it from shared memory.
  const uint32_t smem_base = smem_u32(smem);
  Ranges ahead = seg;                                                // of the places, which are worked out a tile ahead of the copies
  int ahead_tile = 0;
  bool ahead_lives = ahead.next(p);
  if (ahead_lives) ahead_tile = ahead.t0;
  auto advance = [&] {
    if (!ahead_lives || ++ahead_tile < ahead.t1) return;
    ahead_lives = ahead.next(p);
    ahead_tile = ahead.t0;
  };
  auto ahead_drafted = [&] { return ahead_tile + 1 == ahead.tiles; };
  // the page of this thread's token, -1 where there is none
  auto look_up = [&] {
    const int j = ahead_tile * kTile + tid;
    return ahead_lives && !ahead_drafted() && j < ahead.length ? a.page_table[ahead.b * a.page_table_stride + (int)((unsigned long long)j * p.page_magic >> p.page_shift)] : -1;
  };
  int key_scale = -1, value_scale = -1;                              // exponents + 127 of this thread's token of the tile that is copied next, -1: it is not seen
  auto put_place = [&](int page, int parity) {
    if (!ahead_lives) return;
    const int g = ahead.item / p.parts;
    const uint8_t *k = nullptr, *v = nullptr;
    key_scale = value_scale = -1;
    if (ahead_drafted()) {
      if (tid < a.tokens) {
        k = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.k) + ahead.b * a.k_stride[0] + tid * a.k_stride[1] + g * a.k_stride[2]);
        v = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.v) + ahead.b * a.v_stride[0] + tid * a.v_stride[1] + g * a.v_stride[2]);
      }
    } else {
      const int j = ahead_tile * kTile + tid;
      if (j < ahead.length) {
        if ((unsigned)page < (unsigned)a.pages) {
          const int slot = j - (int)((unsigned long long)j * p.page_magic >> p.page_shift) * a.page_size;
          k = static_cast<const uint8_t*>(a.k_cache) + page * a.k_cache_stride[0] + slot * a.k_cache_stride[1] + g * a.k_cache_stride[2];
          v = static_cast<const uint8_t*>(a.v_cache) + page * a.v_cache_stride[0] + slot * a.v_cache_stride[1] + g * a.v_cache_stride[2];
          key_scale = static_cast<const uint8_t*>(sc.k_scales)[page * sc.k_scales_stride[0] + slot * sc.k_scales_stride[1] + g * sc.k_scales_stride[2]];
          value_scale = static_cast<const uint8_t*>(sc.v_scales)[page * sc.v_scales_stride[0] + slot * sc.v_scales_stride[1] + g * sc.v_scales_stride[2]];
        } else {
          flags[0] = 1;
        }
      }
    }
    places[parity * 2 * kTile + tid] = k;
    places[parity * 2 * kTile + kTile + tid] = v;
  };
  auto copy = [&](int stage, int parity, bool drafted) {
    const uint32_t dst = smem_base + stage * kStageBytes;
    const uint8_t** from = places + parity * 2 * kTile;
    if (drafted) {
      const int chunk = tid % kWide;
      for (int row = tid / kWide; row < a.tokens; row += kThreads / kWide) {
        const uint32_t to = dst + row * 2 * D + ((chunk ^ (row & 7)) * 16);
        copy16(to, from[row] + chunk * 16, 16);
        copy16(to + kTileBytes, from[kTile + row] + chunk * 16, 16);
      }
      return;
    }
    const int chunk = tid % kChunks;
#pragma unroll
    for (int i = 0; i < kTile / kRowsPerPass; ++i) {
      const int row = tid / kChunks + i * kRowsPerPass;
      const uint8_t *k = from[row], *v = from[kTile + row];
      const uint32_t to = dst + row * D + ((chunk ^ swizzle<D>(row)) * 16);
      copy16(to, k ? k + chunk * 16 : static_cast<const uint8_t*>(a.q), k ? 16 : 0);
      copy16(to + kTileBytes, v ? v + chunk * 16 : static_cast<const uint8_t*>(a.q), v ? 16 : 0);
    }
  };
  // a token that is not seen: any score becomes minus infinity, a weight of zero
  auto put_constants = [&](int stage, int k, int v) {
    key_by[stage * kTile + tid] = k < 0 ? 0.f : power_of_two(k - 127) * p.scale_log2;
    value_by[stage * kTile + tid] = v < 0 ? make_float2(-INFINITY, 0.f) : make_float2((float)(v - 127), power_of_two(127 - v));
  };
  put_place(look_up(), 0);
#pragma unroll 1
  for (int s = 0; s < kStages - 1; ++s) {
    __syncthreads();
    const bool live = ahead_lives, drafted = live && ahead_drafted();
    if (live) copy(s, s & 1, drafted);
    copies_commit();
    if (live && !drafted) put_constants(s, key_scale, value_scale);
    advance();
    put_place(look_up(), (s + 1) & 1);
  }

  const int quad = lane >> 2, col = lane & 3;                        // this thread's rows quad and quad + 8; tokens 2 col and 2 col + 1 of 8, values 4 col .. 4 col + 3 of 16
  int stage = 0, turn = (kStages - 1) & 1;                           // turn: of the places
#pragma unroll 1
  while (seg.next(p)) {
    const int g = seg.item / p.parts, row0 = seg.item % p.parts * kRowTile, rows = min(p.rows - row0, kRowTile);
    // ---- new rows: queries and masks
    uint32_t q[D / 16][4];
    float o[D / 16][2][4], top[2], total[2], row_by[2];              // sums: [16 values][even and odd ones][row, two values]
    unsigned long long mask[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row_warp * 16 + quad + 8 * h;
      mask[h] = 0;
      const T* src = nullptr;
      if (r < rows) {
        const int t = (row0 + r) / p.group, head = g * p.group + (row0 + r - t * p.group);
        mask[h] = mask_of(p, seg.b, t);
        src = static_cast<const T*>(a.q) + seg.b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2];
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint2 four = src ? *reinterpret_cast<const uint2*>(src + 16 * i + 4 * col) : make_uint2(0u, 0u);
        q[i][h] = four.x;
        q[i][2 + h] = four.y;
      }
      row_by[h] = 1.f;
      if constexpr (!kHalf) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            most = fmaxf(most, fmaxf(finite_magnitude(Half16<T>::value((uint16_t)q[i][e + h])), finite_magnitude(Half16<T>::value((uint16_t)(q[i][e + h] >> 16)))));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int x = exponent_for_half(most);
        const float down = power_of_two(-x);
        row_by[h] = power_of_two(x);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            q[i][e + h] = Half16<half>::pack(Half16<T>::value((uint16_t)q[i][e + h]) * down, Half16<T>::value((uint16_t)(q[i][e + h] >> 16)) * down);
      }
      top[h] = -INFINITY;
      total[h] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][0][e] = o[i][1][e] = 0.f;
    bool odd = false;                                                // infinities or NaN among the drafted values
#pragma unroll 1
    for (int tile = seg.t0; tile < seg.t1; ++tile) {
      copies_wait<kStages - 2>();
      __syncthreads();
      const int refilled = (stage + kStages - 1) % kStages;
      const bool live = ahead_lives, copies_drafted = live && ahead_drafted();
      if (live) copy(refilled, turn, copies_drafted);
      copies_commit();
      const int copied_key_scale = key_scale, copied_value_scale = value_scale;
      advance();
      const int page = look_up();
      turn ^= 1;

      const uint32_t tile_keys = smem_base + stage * kStageBytes, tile_values = tile_keys + kTileBytes;
      const bool drafted = tile + 1 == seg.tiles;
      float s[kMine / 8][4];
      int first = key_warp * kMine, mine = kMine;                    // this warp's tokens of the tile
      if (drafted) {
        // ---- drafted tokens: fp16 with a power of two each; of the values the even ones of 16 before the odd ones, which is how E4M3 values come apart below.
        // Infinities and NaN of values must not meet a weight of zero: they are zero here, and added to the rows that see them at the end.
        first = key_warp * kMyDrafted;
        mine = min(max((a.tokens - first + 15) & ~15, 0), kMyDrafted);
        const int padded = (a.tokens + 15) & ~15;
        bool mine_odd = false;
#pragma unroll 1
        for (int i0 = 0; i0 < 2 * padded * kChunks; i0 += kThreads) {
          const int i = i0 + tid, row = i / kChunks % padded, part = i % kChunks;
          const bool is_value = i / kChunks >= padded, there = i < 2 * padded * kChunks && row < a.tokens;
          const uint32_t at = (is_value ? tile_values : tile_keys) + row * 2 * D;
          const uint32_t lo = at + (((2 * part) ^ (row & 7)) * 16), hi = at + (((2 * part + 1) ^ (row & 7)) * 16);
          uint32_t w[8] = {};
          if (there) {
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(lo) : "memory");
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "r"(hi) : "memory");
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
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fmaxf(finite_magnitude(Half16<T>::value((uint16_t)w[e])), finite_magnitude(Half16<T>::value((uint16_t)(w[e] >> 16)))));
#pragma unroll
            for (int d = 1; d < kChunks; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            x = exponent_for_half(most);
            const float down = power_of_two(-x);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = Half16<half>::pack(Half16<T>::value((uint16_t)w[e]) * down, Half16<T>::value((uint16_t)(w[e] >> 16)) * down);
          }
          if (i < 2 * padded * kChunks) {
            if (is_value) {
              const uint32_t even[4] = {prmt(w[0], w[1], 0x5410), prmt(w[2], w[3], 0x5410), prmt(w[4], w[5], 0x5410), prmt(w[6], w[7], 0x5410)};
              const uint32_t uneven[4] = {prmt(w[0], w[1], 0x7632), prmt(w[2], w[3], 0x7632), prmt(w[4], w[5], 0x7632), prmt(w[6], w[7], 0x7632)};
#pragma unroll
              for (int e = 0; e < 4; ++e) { w[e] = even[e]; w[4 + e] = uneven[e]; }
              if (part == 0) value_by[stage * kTile + row] = make_float2((float)x, power_of_two(-x));
            } else if (part == 0) {
              key_by[stage * kTile + row] = power_of_two(x) * p.scale_log2;
            }
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(lo), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(hi), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
          }
        }
        odd = __syncthreads_or(mine_odd);
      }
      const int tokens8 = mine / 8;                                  // (a warp without drafted tokens has nothing to do)

      // ---- scores of this warp's tokens
      const float* keys_by = key_by + stage * kTile + first;
      const float2* values_by = value_by + stage * kTile + first;
#pragma unroll
      for (int i = 0; i < kMine / 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = drafted ? -INFINITY : 0.f;
      }
      if (!drafted) {
#pragma unroll
        for (int i = 0; i < kMine / 8; ++i) {
          const int row = first + i * 8 + (lane & 7);
#pragma unroll
          for (int d = 0; d < D / 64; ++d) {
            uint32_t k[4];
            ldsm(k, tile_keys + row * D + (((d * 4 + (lane >> 3)) ^ swizzle<D>(row)) * 16));
#pragma unroll
            for (int c = 0; c < 4; ++c) Mma<half>::run(s[i], q[4 * d + c], halves_of(k[c]), halves_of(k[c] >> 16));
          }
          const float2 by = *reinterpret_cast<const float2*>(keys_by + i * 8 + 2 * col);
          const float4 add = *reinterpret_cast<const float4*>(values_by + i * 8 + 2 * col);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kHalf ? s[i][e] : s[i][e] * row_by[e >> 1], e & 1 ? by.y : by.x, e & 1 ? add.z : add.x);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kMyDrafted / 8; ++i) {
          if (i >= tokens8) break;
          const int row = first + i * 8 + quad;
          float x[4] = {};
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t b0, b1;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(tile_keys + row * 2 * D + (((2 * d + (col >> 1)) ^ (row & 7)) * 16) + (col & 1) * 8) : "memory");
            Mma<half>::run(x, q[d], b0, b1);
          }
          const float2 by = *reinterpret_cast<const float2*>(keys_by + i * 8 + 2 * col);
          const float4 add = *reinterpret_cast<const float4*>(values_by + i * 8 + 2 * col);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = first + i * 8 + 2 * col + (e & 1);
            const bool sees = t < a.tokens && (mask[e >> 1] >> t & 1);
            s[i][e] = sees ? fmaf(kHalf ? x[e] : x[e] * row_by[e >> 1], e & 1 ? by.y : by.x, e & 1 ? add.z : add.x) : -INFINITY;
          }
        }
      }

      // ---- running maximum and sum; weights in fp16 for the second product
      float keep[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = top[h];
#pragma unroll
        for (int i = 0; i < kMine / 8; ++i) m = fmaxf(m, fmaxf(s[i][2 * h], s[i][2 * h + 1]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float base = m == -INFINITY ? 0.f : m;                   // nothing seen so far
        keep[h] = exp2_approx(top[h] - base);
        top[h] = m;
        total[h] *= keep[h];
#pragma unroll
        for (int i = 0; i < kMine / 8; ++i) {
          if (drafted && i >= tokens8) break;
          const float4 add = *reinterpret_cast<const float4*>(values_by + i * 8 + 2 * col);
#pragma unroll
          for (int e = 2 * h; e < 2 * h + 2; ++e) {
            s[i][e] = exp2_approx(s[i][e] - base);
            total[h] = fmaf(s[i][e], e & 1 ? add.w : add.y, total[h]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[i][0][e] *= keep[e >> 1];
          o[i][1][e] *= keep[e >> 1];
        }

      // ---- weights times values
#pragma unroll
      for (int k = 0; k < kMine / 16; ++k) {
        if (drafted && 2 * k >= tokens8) break;
        const uint32_t w[4] = {Half16<half>::pack(s[2 * k][0], s[2 * k][1]), Half16<half>::pack(s[2 * k][2], s[2 * k][3]),
                               Half16<half>::pack(s[2 * k + 1][0], s[2 * k + 1][1]), Half16<half>::pack(s[2 * k + 1][2], s[2 * k + 1][3])};
        const int row = first + k * 16 + (lane & 15);
        if (!drafted) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t v[4];
            ldsm_t(v, tile_values + row * D + (((2 * i + (lane >> 4)) ^ swizzle<D>(row)) * 16));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // two tokens' values 2n and 2n + 1 -> the two tokens' values 2n, then those 2n + 1
              const uint32_t x = prmt(v[2 * c], 0, 0x3120), y = prmt(v[2 * c + 1], 0, 0x3120);
              Mma<half>::run(o[2 * i + c][0], w, halves_of(x), halves_of(y));
              Mma<half>::run(o[2 * i + c][1], w, halves_of(x >> 16), halves_of(y >> 16));
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t v[4];
            ldsm_t(v, tile_values + row * 2 * D + (((2 * i + (lane >> 4)) ^ (row & 7)) * 16));
            Mma<half>::run(o[i][0], w, v[0], v[1]);
            Mma<half>::run(o[i][1], w, v[2], v[3]);
          }
        }
      }
      stage = (stage + 1) % kStages;

      if (live && !copies_drafted) put_constants(refilled, copied_key_scale, copied_value_scale);
      put_place(page, turn);
    }

    // ---- the end of this CTA's keys for these rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      total[h] += __shfl_xor_sync(0xffffffffu, total[h], 1);
      total[h] += __shfl_xor_sync(0xffffffffu, total[h], 2);
    }
    // the warps that shared the keys pool their sums, the first one adds them up
    if ((lane & 3) == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        stats[warp * 32 + quad + 8 * h] = top[h];
        stats[warp * 32 + 16 + quad + 8 * h] = total[h];
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float* of = stats + row_warp * kKeyWarps * 32 + quad + 8 * h;
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kKeyWarps; ++w) m = fmaxf(m, of[w * 32]);
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < kKeyWarps; ++w) sum += of[w * 32 + 16] * exp2_approx(of[w * 32] - base);
      const float by = exp2_approx(top[h] - base);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 2 * h; e < 2 * h + 2; ++e) {
          o[i][0][e] *= by;
          o[i][1][e] *= by;
        }
      top[h] = m;
      total[h] = sum;
    }
    // four neighbouring values of a row
    auto four_of = [&](int i, int h) { return make_float4(o[i][0][2 * h], o[i][1][2 * h], o[i][0][2 * h + 1], o[i][1][2 * h + 1]); };
    auto add_four = [&](int i, int h, const float4& x) {
      o[i][0][2 * h] += x.x;
      o[i][1][2 * h] += x.y;
      o[i][0][2 * h + 1] += x.z;
      o[i][1][2 * h + 1] += x.w;
    };
    if (kKeyWarps == 4 && rows <= 4) {
      // there is room for the rows of all warps at once
      float4* place = reinterpret_cast<float4*>(pool) + quad * (D / 4) + col;                       // [warp - 1][row][4 values]
      if (key_warp > 0 && quad < rows) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) place[(key_warp - 1) * D + i * 4] = four_of(i, 0);
      }
      __syncthreads();
      if (key_warp == 0 && quad < rows) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int w = 0; w < 3; ++w) add_four(i, 0, place[w * D + i * 4]);
      }
      __syncthreads();
    } else {
      float4* place = reinterpret_cast<float4*>(pool) + (row_warp * (kKeyWarps - 1) * 16 + quad) * 8 + col;      // [row warp][warp - 1][16 rows][8 times 4 values]
#pragma unroll
      for (int part = 0; part < D / 32; ++part) {
        if (key_warp > 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) place[((key_warp - 1) * 16 + 8 * h) * 8 + i * 4] = four_of(part * 2 + i, h);
        }
        __syncthreads();
        if (key_warp == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int w = 0; w < kKeyWarps - 1; ++w) add_four(part * 2 + i, h, place[(w * 16 + 8 * h) * 8 + i * 4]);
        }
        __syncthreads();
      }
    }
    const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
    if (whole) {
      if (key_warp == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = row_warp * 16 + quad + 8 * h;
          if (r < rows) {
            // padding, and rows that see nothing, are zero
            const bool none = mask[h] == 0 || total[h] == 0.f;
            const float f = 1.f / total[h];
            T* out = out_row<T>(p, seg.b, g, row0 + r) + 4 * col;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const float4 x = four_of(i, h);
              float v[4] = {x.x * f, x.y * f, x.z * f, x.w * f};
              if (odd) add_odd_values<T>(p, seg.b, g, row0 + r, 16 * i + 4 * col, v);
              *reinterpret_cast<uint2*>(out + 16 * i) = none ? make_uint2(0u, 0u) : make_uint2(Half16<T>::pack(v[0], v[1]), Half16<T>::pack(v[2], v[3]));
            }
          }
        }
      }
    } else {
      // a partial: the slot of a range's first rows, or that of its last ones
      float* slot = p.partials + (size_t)(2 * cta + (seg.t0 == 0 ? 1 : 0)) * kSlot;
      if (key_warp == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = row_warp * 16 + quad + 8 * h;
          if (r < rows) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float4*>(slot + r * D + i * 16 + col * 4) = four_of(i, h);
            if ((lane & 3) == 0) {
              slot[kRowTile * D + r] = top[h];
              slot[kRowTile * (D + 1) + r] = total[h];
            }
          }
        }
      }
      if (tid == 0) reinterpret_cast<int*>(slot)[kRowTile * (D + 2)] = odd;
      const int first_cta = seg.t0 == 0 ? cta : cta_of(units, ctas, seg.unit + p.overhead);
      const int last_cta = cta_of(units, ctas, seg.unit + p.overhead + seg.tiles - 1);
      const Joining join(first_cta, last_cta, cta, few_rows_join_step(last_cta - first_cta + 1));
      join_rows<T, D, kRowTile, true>(p, seg.b, g, row0, rows, join, cta, flags + 1);
    }
  }
  copies_wait<0>();
  __syncthreads();
  if (tid == 0 && flags[0] && p.status) atomicExch(p.status, FP6M_ERR_BAD_ARG);
}

template <class T, int D, int kRowTile>
cudaError_t launch_tile(const Fp8Params& p, int ctas, cudaStream_t stream) {
  constexpr int bytes = kStages * (2 * kTile * D + kTile * 12) + kPoolFloats * 4 + 4 * 32 * 4 + 4 * kTile * 8 + sizeof(Plan) + 16;
  cudaError_t e = allow_shared_memory<tree_attention_fp8_kernel<T, D, kRowTile>>(bytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(tree_attention_fp8_kernel<T, D, kRowTile>, dim3(ctas), dim3(kThreads), bytes, stream, p);
}
template <class T>
cudaError_t launch_fp8(Fp8Params p, int ctas, cudaStream_t stream) {
  const bool few = p.tree.rows <= 16;
  p.tree.row_tiles = p.tree.parts = few ? 1 : (p.tree.rows + 31) / 32;
  if (p.tree.a.head_dim == 64) return few ? launch_tile<T, 64, 16>(p, ctas, stream) : launch_tile<T, 64, 32>(p, ctas, stream);
  return few ? launch_tile<T, 128, 16>(p, ctas, stream) : launch_tile<T, 128, 32>(p, ctas, stream);
}

int fp8_ctas(int sms) {
  const int want = sms > 0 ? 2 * sms : kMaxCtas;
  return want < kMaxCtas ? want : kMaxCtas;
}

}  // namespace

extern "C" {

size_t fp6m_tree_attention_fp8_scratch_bytes(int sms) { return kCounterBytes + (size_t)fp8_ctas(sms) * 2 * slot_floats<128, 32, true>() * sizeof(float); }

int fp6m_tree_attention_fp8(const fp6m_tree_attention_args* args, const fp6m_cache_scales* scales, void* scratch, size_t scratch_bytes, int dev, void* stream, int* status_dev) {
  if (!args || !scales) return FP6M_ERR_BAD_ARG;
  Fp8Params p;
  p.scales = *scales;
  const int rc = check_tree_args(*args, 16, scratch);
  if (rc != FP6M_OK || args->batch == 0 || args->tokens == 0 || args->heads == 0) return rc;
  if (args->max_pages > 0 && (!scales->k_scales || !scales->v_scales)) return FP6M_ERR_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (scales->k_scales_stride[i] < 0 || scales->v_scales_stride[i] < 0) return FP6M_ERR_BAD_ARG;
  DeviceGuard guard(dev);
  const int sms = sm_count(dev);
  if (sms <= 0) return cuda_fail(cudaGetLastError(), "cudaDeviceGetAttribute");
  if (scratch_bytes < fp6m_tree_attention_fp8_scratch_bytes(sms)) return FP6M_ERR_SCRATCH;
  p.tree = tree_params(*args, scratch, kCounterBytes, status_dev);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = args->type == FP6M_TYPE_F16 ? launch_fp8<half>(p, fp8_ctas(sms), st) : launch_fp8<__nv_bfloat16>(p, fp8_ctas(sms), st);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "tree_attention_fp8 launch");
}

}  // extern "C"
