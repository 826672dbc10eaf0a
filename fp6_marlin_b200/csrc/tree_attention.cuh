// Shared by the kernels of attention over a paged cache (tree_attention.cu, tree_attention_tc5.cu, tree_attention_fp8.cu).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp6m.h"
#include "device_utils.cuh"
#include "host_common.h"

namespace fp6m {

constexpr int kKeys = 64;                // keys per tile
constexpr int kMaxTreeCtas = 512;
constexpr int kCounterBytes = kMaxTreeCtas * 2 * 3 * 4;

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
// With a cache in 8 bits: 21.3 / 35.5; 24.7 / 34.3; up to 6144 148 / 195 (bf16 154 / 241); 36.6 / 54.3; one sequence of 32768, 4 tokens, 41.9 / 50.8.
constexpr int kFewRows = 32;
size_t tree_tc5_partial_bytes(int sms);
cudaError_t launch_tree_tc5(TreeParams p, const fp6m_cache_scales* scales, int sms, cudaStream_t stream);      // scales: of a cache in 8 bits, or null

// Addresses and strides of a tensor that is read or written sixteen bytes at a time, `of` elements.
template <int kStrides>
bool rows_aligned(const void* p, const long long (&strides)[kStrides], int of) {
  bool ok = p && aligned16(p);
  for (long long s : strides) ok = ok && s >= 0 && s % of == 0;
  return ok;
}
// What the entries check before they touch the GPU; `cache_of`: values of the cache in sixteen bytes.
inline int check_tree_args(const fp6m_tree_attention_args& a, int cache_of, const void* scratch) {
  if (a.batch < 0 || a.tokens < 0 || a.heads < 0 || (a.type != FP6M_TYPE_F16 && a.type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (a.tokens > 64 || (a.head_dim != 64 && a.head_dim != 128)) return FP6M_ERR_PROB_SHAPE;
  if (a.batch == 0 || a.tokens == 0 || a.heads == 0) return FP6M_OK;
  if (a.kv_heads <= 0 || a.heads % a.kv_heads) return FP6M_ERR_PROB_SHAPE;
  // (pages are looked up in blocks of up to 2048 tokens, two of them ahead, so tokens stay that far from 2^31)
  if (a.max_pages < 0 || a.pages < 0 || a.page_size <= 0 || (long long)a.max_pages * a.page_size > 0x7fff0000ll) return FP6M_ERR_PROB_SHAPE;
  if ((long long)a.tokens * a.heads > 0xffffffll) return FP6M_ERR_PROB_SHAPE;
  if (!rows_aligned(a.q, a.q_stride, 8) || !rows_aligned(a.k, a.k_stride, 8) || !rows_aligned(a.v, a.v_stride, 8) || !rows_aligned(a.out, a.out_stride, 8)) return FP6M_ERR_BAD_ARG;
  if (!a.lengths || !a.tree || a.tree_stride < 0 || !scratch || !aligned16(scratch)) return FP6M_ERR_BAD_ARG;
  if (a.max_pages > 0 && (!rows_aligned(a.k_cache, a.k_cache_stride, cache_of) || !rows_aligned(a.v_cache, a.v_cache_stride, cache_of) || !a.page_table || a.page_table_stride < 0)) return FP6M_ERR_BAD_ARG;
  return FP6M_OK;
}
// n / divisor = n * magic >> shift, exact for n < 2^31
inline void division_by(int divisor, unsigned long long* magic, int* shift) {
  int log2 = 0;
  while ((1ll << log2) < divisor) ++log2;
  *shift = 31 + log2;
  *magic = ((1ull << *shift) + divisor - 1) / divisor;
}
inline TreeParams tree_params(const fp6m_tree_attention_args& a, void* scratch, size_t counter_bytes, int* status_dev) {
  TreeParams p = {};
  p.a = a;
  p.group = a.heads / a.kv_heads;
  p.rows = a.tokens * p.group;
  p.row_tiles = p.parts = 1;
  p.overhead = 4;
  division_by(a.page_size, &p.page_magic, &p.page_shift);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  if (p.scale_log2 == 0.f) p.scale_log2 = 1e-37f;      // a masked score of minus infinity stays that
  p.arrived = static_cast<unsigned int*>(scratch);
  p.partials = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + counter_bytes);
  p.status = status_dev;
  return p;
}

#ifdef __CUDACC__

// The mask of token t of sequence b: the drafted tokens that it sees (bits behind the last of them mean nothing), 0 for padding.
__device__ __forceinline__ unsigned long long mask_of(const TreeParams& p, int b, int t) { return p.a.tree[b * p.a.tree_stride + t]; }
__device__ __forceinline__ int length_of(const TreeParams& p, int b) {
  const int n = p.a.lengths[b], most = p.a.max_pages * p.a.page_size;
  return n < 0 ? 0 : n > most ? most : n;
}

// How many tiles a sequence's keys make.  Here: of 64 keys, the drafted tokens behind the cached ones in the same tile.
struct TilesTogether {
  static __device__ __forceinline__ int of(const TreeParams& p, int length) { return (int)(((long long)length + p.a.tokens + kKeys - 1) / kKeys); }
};

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
template <class Tiles = TilesTogether>
__device__ __forceinline__ void make_plan(const TreeParams& p, Plan* plan, int least, int slack) {
  const int lane = threadIdx.x & 31, cta = blockIdx.x, grid = gridDim.x;
  const long long items = (long long)p.a.kv_heads * p.parts;
  long long units = 0;
  int longest = 0;
  for (int b = lane; b < p.a.batch; b += 32) {
    const int size = Tiles::of(p, length_of(p, b)) + p.overhead;
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
      plan->count = Tiles::of(p, plan->length) + p.overhead;
      plan->at = (cta % (int)items) * plan->count;
      plan->start = 0;
    }
    return;
  }
  const long long first = cta < ctas ? range_start(units, ctas, cta) : units;
  long long before = 0;
  for (int b0 = 0; b0 < p.a.batch; b0 += 32) {
    const int b = b0 + lane, length = b < p.a.batch ? length_of(p, b) : 0;
    const long long mine = b < p.a.batch ? (Tiles::of(p, length) + p.overhead) * items : 0;
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
template <class Tiles>
struct SegmentsOf {
  int b, length, tiles, item, t0, t1;    // the segment
  long long unit;                        // where its item starts
  int at;                                // unit inside the item of what follows
  long long left;                        // units that follow
  __device__ __forceinline__ SegmentsOf(const TreeParams& p, const Plan& plan) {
    b = plan.b;
    length = plan.length;
    tiles = Tiles::of(p, length);
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
          tiles = Tiles::of(p, length);
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
using Segments = SegmentsOf<TilesTogether>;

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
// four bytes
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
// arrives once this thread's copies so far have landed
__device__ __forceinline__ void copies_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// p.run tokens of a head, a box's values from x on: value x, head, slot, page.  x is 0 or 64 values of 16 bits (128 bytes), so the copy starts on a 16-byte boundary.
__device__ __forceinline__ void tma_load_run(uint32_t dst, const CUtensorMap* map, int x, int head, int slot, int page, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(x), "r"(head), "r"(slot), "r"(page), "r"(bar) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// the lower and the upper two of four E4M3 values in fp16 (exact)
__device__ __forceinline__ uint32_t halves_of(uint32_t four) {
  uint32_t h;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(h) : "r"(four));
  return h;
}
__device__ __forceinline__ uint32_t upper_halves_of(uint32_t four) {
  uint32_t h;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(h) : "r"(four));
  return h;
}
constexpr float kGrowth = 8.f;           // log2 of the growth of a maximum that is let pass: weights are relative to an older one until then
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

// ---- for the kernels whose rows are few (tree_attention.cu, tree_attention_fp8.cu)
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

#endif  // __CUDACC__

}  // namespace fp6m
