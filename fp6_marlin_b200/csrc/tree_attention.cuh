// Shared by the kernels of attention over a paged cache (tree_attention.cu, tree_attention_tc5.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp6m.h"

namespace fp6m {

constexpr int kKeys = 64;                // keys per tile

struct TreeParams {
  fp6m_tree_attention_args a;
  int group, rows;                       // heads of queries per head of keys; rows of a head of keys
  int row_tiles, parts;                  // the tiles that the rows are cut into, and the items they make (one or two tiles each)
  int overhead;                          // what the rows of an item cost besides their key tiles, in key tiles
  unsigned long long page_magic;         // division by the page size: n * magic >> shift, exact for n < 2^31
  int page_shift;
  int run;                               // tokens of a page that one TMA copy brings (0: none does)
  float scale_log2;                      // scale * log2(e): the softmax is computed in powers of two
  unsigned int* arrived;                 // [CTA][row tile of two][3] contributors that have left their partial, see Joining
  float* partials;
  int* status;
};

// tree_attention_tc5.cu: more rows than kFewRows.  us for 20 to 32 rows, few / many: 8 x 4 tokens, 32 heads over 4, 2048 cached 27.8 / 26.4;
// 2 x 3, 64 over 8, 8192: 34.9 / 36.7; 64 x 4, 64 over 8, up to 4096: 114.2 / 114.7; 16 x 5, 32 over 8, up to 4000: 41.4 / 44.4.
constexpr int kFewRows = 32;
size_t tree_tc5_partial_bytes(int sms);
cudaError_t launch_tree_tc5(TreeParams p, int sms, cudaStream_t stream);

#ifdef __CUDACC__

// The mask of token t of sequence b: the drafted tokens that it sees (bits behind the last of them mean nothing), 0 for padding.
__device__ __forceinline__ unsigned long long mask_of(const TreeParams& p, int b, int t) { return p.a.tree[b * p.a.tree_stride + t]; }
__device__ __forceinline__ int length_of(const TreeParams& p, int b) {
  const int n = p.a.lengths[b], most = p.a.max_pages * p.a.page_size;
  return n < 0 ? 0 : n > most ? most : n;
}
__device__ __forceinline__ int tiles_of(const TreeParams& p, int length) { return (int)(((long long)length + p.a.tokens + kKeys - 1) / kKeys); }

// The work is a line of units: for every sequence, head of keys and row tile (an item: one row tile, or two) `overhead` units, then one for each key tile.
// CTAs take equal ranges of it.
__device__ __forceinline__ long long range_start(long long units, int ctas, int cta) { return units * cta / ctas; }
__device__ __forceinline__ int cta_of(long long units, int ctas, long long unit) {
  int c = (int)(unit * ctas / units);
  while (c + 1 < ctas && range_start(units, ctas, c + 1) <= unit) ++c;
  while (range_start(units, ctas, c) > unit) --c;
  return c;
}

// How the units are shared out, and where this CTA starts: worked out by one warp, in shared memory.
struct Plan {
  long long units, start, count;         // in all; this CTA's first and how many
  long long at;                          // its first unit, from the start of the sequence on
  int ctas, b, length, apart;            // CTAs that work; the sequence of the first unit, and its length; apart: an item per CTA
};
// `least`: units of a CTA, fewer cost less than joining what more CTAs leave; `slack`: what that joining takes, in key tiles: where there
// are CTAs enough for an item each, and the longest item is not that much longer than an equal share, every CTA gets one item.
__device__ __forceinline__ void make_plan(const TreeParams& p, Plan* plan, int least, int slack) {
  const int lane = threadIdx.x & 31, cta = blockIdx.x, grid = gridDim.x;
  const long long items = (long long)p.a.kv_heads * p.parts;
  long long units = 0;
  int longest = 0;
  for (int b = lane; b < p.a.batch; b += 32) {
    const int size = tiles_of(p, length_of(p, b)) + p.overhead;
    units += size * items;
    longest = max(longest, size);
  }
  for (int o = 16; o; o >>= 1) {
    units += __shfl_xor_sync(0xffffffffu, units, o);
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  const int ctas = (long long)grid < units / least ? grid : max((int)(units / least), 1);
  const bool apart = items * p.a.batch <= grid && longest - units / ctas <= slack;
  if (apart) {
    if (lane == 0) {
      plan->ctas = (int)items * p.a.batch;
      plan->apart = 1;
      plan->b = min(cta / (int)items, p.a.batch - 1);
      plan->length = length_of(p, plan->b);
      plan->units = units;
      plan->count = tiles_of(p, plan->length) + p.overhead;
      plan->at = (cta % (int)items) * plan->count;
      plan->start = 0;
    }
    return;
  }
  const long long first = cta < ctas ? range_start(units, ctas, cta) : units;
  long long before = 0;
  for (int b0 = 0; b0 < p.a.batch; b0 += 32) {
    const int b = b0 + lane, length = b < p.a.batch ? length_of(p, b) : 0;
    const long long mine = b < p.a.batch ? (tiles_of(p, length) + p.overhead) * items : 0;
    long long upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (first >= before + upto - mine && first < before + upto) {
      plan->at = first - (before + upto - mine);
      plan->b = b;
      plan->length = length;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    if (before > first) break;
  }
  if (lane == 0) {
    plan->units = units;
    plan->ctas = ctas;
    plan->apart = 0;
    plan->start = first;
    plan->count = cta < ctas ? range_start(units, ctas, cta + 1) - first : 0;
  }
}

// A CTA's range as a sequence of segments: the key tiles t0 .. t1 - 1 of an item.
struct Segments {
  int b, length, tiles, item, t0, t1;    // the segment
  long long unit;                        // where its item starts
  int at;                                // unit inside the item of what follows
  long long left;                        // units that follow
  __device__ __forceinline__ Segments(const TreeParams& p, const Plan& plan) {
    b = plan.b;
    length = plan.length;
    tiles = tiles_of(p, length);
    const int size = tiles + p.overhead;
    item = (int)(plan.at / size);
    at = (int)(plan.at - (long long)item * size);
    unit = plan.start - at;
    left = plan.count;
  }
  __device__ __forceinline__ bool next(const TreeParams& p) {
    while (left > 0) {
      const int size = tiles + p.overhead;
      if (at == size) {
        at = 0;
        unit += size;
        if (++item == p.a.kv_heads * p.parts) {
          item = 0;
          ++b;
          length = length_of(p, b);
          tiles = tiles_of(p, length);
        }
        continue;
      }
      const int take = left < size - at ? (int)left : size - at;
      t0 = max(at - p.overhead, 0);
      t1 = at + take - p.overhead;
      at += take;
      left -= take;
      if (t1 > t0) return true;
    }
    return false;
  }
};

// How the partials of an item's contributors (the CTAs first .. last) become one: by the contributor that is the last to leave its own, all of them in
// their order - or, where they are many, in groups of `step` first: the last of a group leaves the sum in the slot of its first, and the
// last of those adds up the groups.  Every group has a counter, at its first CTA: [0] the item starts there, [1] it started before
// (a CTA has one such item at most); [2] counts the groups, where the item starts.  Nobody waits, and the order of the sums is the ranges'.
struct Joining {
  int first, count, step, group, size;   // the item's contributors; this CTA's group's first, and how many it has
  __device__ __forceinline__ Joining(int first_cta, int last_cta, int cta, int step_) {
    first = first_cta;
    count = last_cta - first_cta + 1;
    step = step_;
    group = first + (cta - first) / step * step;
    size = min(step, last_cta + 1 - group);
  }
  __device__ __forceinline__ int groups() const { return (count + step - 1) / step; }
  __device__ __forceinline__ unsigned int* group_counter(const TreeParams& p, int which) const { return p.arrived + (group * 2 + which) * 3 + (group == first ? 0 : 1); }
  __device__ __forceinline__ unsigned int* item_counter(const TreeParams& p, int which) const { return p.arrived + (first * 2 + which) * 3 + 2; }
};

// The first value of key (or value) j of a sequence, null where there is none: behind the last one, or in a page that does not exist.
template <class T>
__device__ __forceinline__ const T* place_of(const TreeParams& p, const Segments& s, int g, int j, int page, bool values) {
  const fp6m_tree_attention_args& a = p.a;
  const long long* strides = values ? a.v_cache_stride : a.k_cache_stride;
  if (j < s.length) {
    if ((unsigned)page >= (unsigned)a.pages) return nullptr;
    const int slot = j - (int)((unsigned long long)j * p.page_magic >> p.page_shift) * a.page_size;
    return static_cast<const T*>(values ? a.v_cache : a.k_cache) + page * strides[0] + slot * strides[1] + g * strides[2];
  }
  if (j - s.length >= a.tokens) return nullptr;
  const long long* drafted = values ? a.v_stride : a.k_stride;
  return static_cast<const T*>(values ? a.v : a.k) + s.b * drafted[0] + (j - s.length) * drafted[1] + g * drafted[2];
}
__device__ __forceinline__ int page_of(const TreeParams& p, const Segments& s, int j) {
  return j < s.length ? p.a.page_table[s.b * p.a.page_table_stride + (int)((unsigned long long)j * p.page_magic >> p.page_shift)] : 0;
}

// sixteen bytes, or zeros where `bytes` is 0 (the source is not read then)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T> struct Half16;
template <> struct Half16<half> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) { half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<uint32_t*>(&h); }
  static __device__ __forceinline__ float value(uint16_t bits) { return __half2float(__ushort_as_half(bits)); }
  static constexpr uint32_t kExponent = 0x7c00u;       // all ones: infinite or NaN
  static constexpr uint32_t kMmaFormat = 0;
};
template <> struct Half16<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) { __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<uint32_t*>(&h); }
  static __device__ __forceinline__ float value(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
  static constexpr uint32_t kExponent = 0x7f80u;
  static constexpr uint32_t kMmaFormat = 1;
};
// whether one of the two values is infinite or NaN
template <class T>
__device__ __forceinline__ bool is_odd(uint32_t two) {
  constexpr uint32_t E = Half16<T>::kExponent;
  return (two & E) == E || (two >> 16 & E) == E;
}

#endif  // __CUDACC__

}  // namespace fp6m
