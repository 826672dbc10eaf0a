// Shared by the kernels of attention over a paged cache (tree_attention.cu, tree_attention_tc5.cu, tree_attention_fp8.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp6m.h"
#include "host_common.h"

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

// ---- for the kernels of four warps whose rows are few (tree_attention.cu, tree_attention_fp8.cu) ----

template <class T> struct Mma;
template <> struct Mma<half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// contributors of a group: see Joining
__device__ __forceinline__ int few_rows_join_step(int count) {
  if (count <= 24) return count;
  int step = 8;
  while (step * step < count) step += 8;
  return step;
}
// Where row r of a head of keys goes.
template <class T>
__device__ __forceinline__ T* out_row(const TreeParams& p, int b, int g, int r) {
  const int t = r / p.group, head = g * p.group + (r - t * p.group);
  return static_cast<T*>(p.a.out) + b * p.a.out_stride[0] + t * p.a.out_stride[1] + head * p.a.out_stride[2];
}
// A partial: sums [row][column], maxima, totals, and (kOdd) whether infinities or NaN were met among the drafted values, which are added at the end.
template <int D, int kRowTile, bool kOdd>
constexpr int slot_floats() { return kRowTile * (D + 2) + (kOdd ? 4 : 0); }
// The infinite and NaN values of the drafted tokens that row r sees, added to columns c .. c + N - 1 of its result.
template <class T, int N>
__device__ __forceinline__ void add_odd_values(const TreeParams& p, int b, int g, int r, int c, float (&v)[N]) {
  const unsigned long long mask = mask_of(p, b, r / p.group);
  for (int j = 0; j < p.a.tokens; ++j) {
    if (!(mask >> j & 1)) continue;
    const uint16_t* from = static_cast<const uint16_t*>(p.a.v) + b * p.a.v_stride[0] + j * p.a.v_stride[1] + g * p.a.v_stride[2] + c;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((from[i] & Half16<T>::kExponent) == Half16<T>::kExponent) v[i] += Half16<T>::value(from[i]);
  }
}
// Called by all threads of a CTA that has left its partial of rows row0 .. row0 + rows - 1 of (b, g): the last contributor joins them (see Joining).
template <class T, int D, int kRowTile, bool kOdd>
__device__ __forceinline__ void join_rows(const TreeParams& p, int b, int g, int row0, int rows, const Joining& join, int cta, int* last_flag) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, first_cta = join.first;
  constexpr int kSlot = slot_floats<D, kRowTile, kOdd>();
  // whether this CTA is the last of those that a counter waits for; what the others wrote is visible then
  auto last_at = [&](unsigned int* counter, int others) {
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const bool is_last = atomicAdd(counter, 1u) == (unsigned)others;
      if (is_last) *counter = 0;                               // for the next launch
      *last_flag = is_last;
    }
    __syncthreads();
    const bool is_last = *last_flag != 0;
    __threadfence();
    return is_last;
  };
  auto slot_of = [&](int c) { return p.partials + (size_t)(2 * c + (c == first_cta ? 1 : 0)) * kSlot; };
  // Joins `count` partials, `step` CTAs apart: into the output, or into the first one's slot.  A warp has two rows at a time, a lane four or two columns of
  // each; a lane fetches the maximum and total of one contributor, and eight contributors' sums are on their way together (one after the other took
  // a latency each; 24 rows of 19 contributors: 43 us in all then, 35 now).
  auto add_up = [&](int c0, int count, int step, bool ends) {
    constexpr int V = D / 32, kTogether = 8;
    // (the drafted tokens are the last contributor's)
    const bool odd = kOdd && ends && __ldcg(reinterpret_cast<const int*>(slot_of(first_cta + join.count - 1)) + kRowTile * (D + 2)) != 0;
    for (int r0 = warp; r0 < rows; r0 += 8) {
      float m[2] = {-INFINITY, -INFINITY}, sum[2] = {}, acc[2][V] = {};
      const int of[2] = {r0, r0 + 4 < rows ? r0 + 4 : r0};
      for (int k0 = 0; k0 < count; k0 += 32) {
        const int here = min(count - k0, 32);
        float by[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* from = slot_of(c0 + (k0 + min(lane, here - 1)) * step) + kRowTile * D + of[h];
          const float cm = lane < here ? __ldcg(from) : -INFINITY, ct = lane < here ? __ldcg(from + kRowTile) : 0.f;
          float most = cm;
#pragma unroll
          for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          const float now = fmaxf(m[h], most), base = now == -INFINITY ? 0.f : now, old = exp2_approx(m[h] - base);
          by[h] = exp2_approx(cm - base);
          float part = ct * by[h];
#pragma unroll
          for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
          sum[h] = sum[h] * old + part;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[h][i] *= old;
          m[h] = now;
        }
        for (int j0 = 0; j0 < here; j0 += kTogether) {
          float2 v[kTogether][2][V / 2];
#pragma unroll
          for (int e = 0; e < kTogether; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < V / 2; ++i)
                v[e][h][i] = j0 + e < here ? __ldcg(reinterpret_cast<const float2*>(slot_of(c0 + (k0 + j0 + e) * step) + of[h] * D + lane * V) + i) : make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < kTogether; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f = __shfl_sync(0xffffffffu, by[h], (j0 + e) & 31);
#pragma unroll
              for (int i = 0; i < V / 2; ++i) {
                acc[h][2 * i] = fmaf(v[e][h][i].x, f, acc[h][2 * i]);
                acc[h][2 * i + 1] = fmaf(v[e][h][i].y, f, acc[h][2 * i + 1]);
              }
            }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = r0 + 4 * h;
        if (r >= rows) break;
        if (ends) {
          const bool none = mask_of(p, b, (row0 + r) / p.group) == 0 || sum[h] == 0.f;      // padding, and rows that see nothing, are zero
          const float f = 1.f / sum[h];
          T* out = out_row<T>(p, b, g, row0 + r) + lane * V;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[h][i] *= f;
          if (kOdd && odd) add_odd_values<T>(p, b, g, row0 + r, lane * V, acc[h]);
#pragma unroll
          for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(out + i) = none ? 0u : Half16<T>::pack(acc[h][i], acc[h][i + 1]);
        } else {
          float* to = slot_of(c0);
#pragma unroll
          for (int i = 0; i < V; i += 2) __stcg(reinterpret_cast<float2*>(to + r * D + lane * V + i), make_float2(acc[h][i], acc[h][i + 1]));
          if (lane == 0) {
            __stcg(to + kRowTile * D + r, m[h]);
            __stcg(to + kRowTile * (D + 1) + r, sum[h]);
          }
        }
      }
    }
  };
  // (one loop, so that its code is there once: what runs for the first time takes longer to fetch than to run)
  const bool grouped = join.step < join.count;
  bool ends = !grouped;
#pragma unroll 1
  while (last_at(ends && grouped ? join.item_counter(p, 0) : join.group_counter(p, 0), (ends && grouped ? join.groups() : join.size) - 1)) {
    add_up(ends ? first_cta : join.group, ends && grouped ? join.groups() : join.size, ends && grouped ? join.step : 1, ends);
    if (ends) break;
    ends = true;
  }
}

#endif  // __CUDACC__

}  // namespace fp6m
