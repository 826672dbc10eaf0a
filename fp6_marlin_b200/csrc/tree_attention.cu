// Attention of T drafted tokens of each of B sequences over a paged cache of committed tokens and the drafted tokens themselves.
//
//   o_i = sum_j p_ij v_j,   p_i = softmax_j(scale * q_i . k_j)
//
// over the lengths[b] cached tokens and the drafted tokens j whose bit is set in the mask of i.  A mask of zero marks padding:
// it sees nothing and gives zeros.  The reference has no counterpart; its layer lists (bench.py:53-86) name the products on either side.
//
// The queries that share a head of keys - T tokens times heads / kv_heads heads - are the rows of one product; a sequence's keys
// are its cached tokens followed by its drafted ones, in tiles of 64.  The (sequence, head of keys, row tile, key tile) units
// are cut into equal ranges, one per CTA, so that long and short sequences and few heads load all multiprocessors alike; the
// cut is made on the device, from the lengths, and the launch does not depend on them.  One pass over the keys keeps a
// running maximum and sum per row in fp32.  Rows whose keys are shared by several CTAs are joined by the one that finishes
// last (an arrival counter; nobody waits), in the order of the ranges, so results do not depend on who that is.
//
// This file: up to 32 rows per head of keys, where mma.sync keeps up with memory (rows are padded to 16 or 32, a tile of tcgen05 would have 128) and what counts is
// the time from a key's arrival to its use.  Two CTAs per multiprocessor, three tiles of keys and values on their way in each.  8 x 5 tokens, 32 heads, up to
// 4096 cached, public calls one behind the other: 56 us, 4.8 TB/s, 0.73 of what a copy reaches; bound by the instructions between two tiles (about 1660 cycles a tile and CTA) and
// the tails of CTAs.  One token over 300: 10.6 us where the bytes take 0.8: the plan (2000 cycles), first look-ups and queries (2900), first data
// (1200), two or three tiles, the end (1700).  Figures of both sides of a choice are of replays of a graph.
//
// The weights are rounded once, to the values' type, for the second product (tensor cores take 16 bits; the sum that they are divided by has them unrounded): 2^-8 of
// a weight at most in bf16, 2^-11 in fp16, where weights below 2^-14 of the largest become multiples of 2^-24.
#include "device_utils.cuh"
#include "host_common.h"
#include "tree_attention.cuh"

namespace {

using namespace fp6m;

constexpr int kThreads = 128;
constexpr int kMaxCtas = 512;
// see make_plan.  us with a slack of 4 / 8 / 16: one token over 300, 32 heads 12.9 / 12.2 / 12.2; four over 500 13.4 / 13.3 / 15.6.
// With at least 3 / 6 units per CTA: one token over 1000, 32 heads over 8, 12.9 / 17.0; sixteen over up to 500 13.4 / 15.4; one over 8000 17.9 / 19.1.
constexpr int kLeastUnits = 3, kSlack = 8;
constexpr int kCounterBytes = kMaxCtas * 2 * 3 * 4;
// contributors of a group: see Joining
__device__ __forceinline__ int join_step(int count) {
  if (count <= 24) return count;
  int step = 8;
  while (step * step < count) step += 8;
  return step;
}

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
// kRowTile rows, a warp for every 16 of them; the warps that this leaves share the keys of a tile and pool their sums.
template <class T, int D, int kRowTile>
__global__ void __launch_bounds__(kThreads, 2) tree_attention_kernel(const __grid_constant__ TreeParams p) {
  constexpr int kRowWarps = kRowTile / 16, kKeyWarps = 4 / kRowWarps;
  constexpr int kMine = kKeys / kKeyWarps;                           // keys of a tile that a warp works on
  constexpr int kRowBytes = D * 2, kTileBytes = kKeys * kRowBytes;   // keys or values of a tile
  constexpr int kStages = 3 * 128 / D;
  constexpr int kChunks = D / 8, kRowsPerPass = kThreads / kChunks, kPasses = kKeys / kRowsPerPass;
  constexpr int kPool = D / kRowWarps;                               // columns of the sums that are pooled at a time
  constexpr int kSlot = kRowTile * (D + 2);                          // floats of a partial
  extern __shared__ __align__(128) uint8_t smem[];
  float* pool = reinterpret_cast<float*>(smem + kStages * 2 * kTileBytes);        // [kRowTile][kPool]
  float* stats = pool + kRowTile * kPool;                                          // [warp][2][16]: maxima, totals
  Plan* plan = reinterpret_cast<Plan*>(stats + 4 * 32);
  int* flags = reinterpret_cast<int*>(plan + 1);                                   // [0] a page did not exist, [1] last to arrive
  const T** places = reinterpret_cast<const T**>(flags + 4);                       // [2][128]: where the keys, then the values, of a tile are

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row_warp = warp / kKeyWarps, key_warp = warp % kKeyWarps;
  const fp6m_tree_attention_args& a = p.a;
  if (tid == 0) flags[0] = 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cta = blockIdx.x;
  if (warp == 0) make_plan(p, plan, kLeastUnits, kSlack);
  __syncthreads();
  const long long units = plan->units;
  const int ctas = plan->ctas;
  if (cta >= ctas) return;
  Segments seg(p, *plan);

  // ---- copies of a tile: a row of keys and one of values per token, zeros behind the last.  A thread works out where one row is (the
  // same by all threads that copy a piece of it cost half of the kernel's instructions); the others take it from shared memory.
  const uint32_t smem_base = smem_u32(smem);
  const int load_row = tid / kChunks, chunk = tid % kChunks;
  Segments ahead = seg;                                              // of the places, which are worked out a tile ahead of the copies
  int ahead_tile = 0;
  bool ahead_lives = ahead.next(p);
  if (ahead_lives) ahead_tile = ahead.t0;
  auto advance = [&] {
    if (!ahead_lives || ++ahead_tile < ahead.t1) return;
    ahead_lives = ahead.next(p);
    ahead_tile = ahead.t0;
  };
  const int my_key = tid % kKeys;
  auto look_up = [&] { return ahead_lives ? page_of(p, ahead, ahead_tile * kKeys + my_key) : 0; };
  auto put_place = [&](int page, int parity) {
    const int j = ahead_tile * kKeys + my_key;
    const T* place = ahead_lives ? place_of<T>(p, ahead, ahead.item, j, page, tid >= kKeys) : nullptr;
    if (ahead_lives && !place && j < ahead.length) flags[0] = 1;
    places[parity * kThreads + tid] = place;
  };
  auto copy = [&](int stage, int parity) {
    const uint32_t dst = smem_base + stage * 2 * kTileBytes;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = load_row + i * kRowsPerPass;
      const T *k = places[parity * kThreads + row], *v = places[parity * kThreads + kKeys + row];
      const uint32_t to = dst + row * kRowBytes + ((chunk ^ (row & 7)) * 16);
      copy16(to, k ? k + chunk * 8 : static_cast<const T*>(a.q), k ? 16 : 0);
      copy16(to + kTileBytes, v ? v + chunk * 8 : static_cast<const T*>(a.q), v ? 16 : 0);
    }
  };
  int page = look_up();
  // (the page of the next tile is looked up before the place of this one is worked out: the first two look-ups take one latency)
  auto look_up_next = [&] {
    const Segments before = ahead;
    const int tile_before = ahead_tile;
    const bool lived = ahead_lives;
    advance();
    const int next = look_up();
    ahead = before;
    ahead_tile = tile_before;
    ahead_lives = lived;
    return next;
  };
  int next_page = look_up_next();
  put_place(page, 0);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    __syncthreads();
    const bool live = ahead_lives;
    advance();
    if (s > 0) next_page = look_up();
    if (live) copy(s, s & 1);
    copies_commit();
    put_place(next_page, (s + 1) & 1);
  }

  const int quad = lane >> 2, col = (lane & 3) * 2;                  // this thread's rows quad and quad + 8, columns col and col + 1 of a fragment
  int stage = 0, turn = (kStages - 1) & 1;                           // turn: of the places
#pragma unroll 1
  while (seg.next(p)) {
    const int g = seg.item;
    // ---- new rows: queries and masks
    uint32_t q[D / 16][4];
    float o[D / 8][4], top[2], total[2];
    unsigned long long mask[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row_warp * 16 + quad + 8 * h;
      mask[h] = 0;
      const T* src = nullptr;
      if (r < p.rows) {
        const int t = r / p.group, head = g * p.group + (r - t * p.group);
        mask[h] = mask_of(p, seg.b, t);
        src = static_cast<const T*>(a.q) + seg.b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2];
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        q[i][h] = src ? *reinterpret_cast<const uint32_t*>(src + 16 * i + col) : 0u;
        q[i][2 + h] = src ? *reinterpret_cast<const uint32_t*>(src + 16 * i + 8 + col) : 0u;
      }
      top[h] = -INFINITY;
      total[h] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll 1
    for (int tile = seg.t0; tile < seg.t1; ++tile) {
      copies_wait<kStages - 2>();
      __syncthreads();
      const bool live = ahead_lives;
      advance();
      const int page = look_up();
      if (live) copy((stage + kStages - 1) % kStages, turn);
      copies_commit();
      turn ^= 1;

      // ---- scores of this warp's keys
      const uint32_t keys = smem_base + stage * 2 * kTileBytes + key_warp * kMine * kRowBytes, values = keys + kTileBytes;
      float s[kMine / 8][4];
#pragma unroll
      for (int i = 0; i < kMine / 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
        const int row = i * 8 + (lane & 7);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          uint32_t k[4];
          ldsm(k, keys + row * kRowBytes + (((d * 4 + (lane >> 3)) ^ (row & 7)) * 16));
          Mma<T>::run(s[i], q[2 * d], k[0], k[1]);
          Mma<T>::run(s[i], q[2 * d + 1], k[2], k[3]);
        }
      }
      const int j0 = tile * kKeys + key_warp * kMine;               // this warp's first key
      const bool drafted = tile * kKeys + kKeys > seg.length;        // the tile holds drafted tokens, or the end
      const bool hidden = flags[0] != 0;                               // a page of this CTA's tiles did not exist
#pragma unroll
      for (int i = 0; i < kMine / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] *= p.scale_log2;
      if (drafted) {
#pragma unroll
        for (int i = 0; i < kMine / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = j0 + i * 8 + col + (e & 1) - seg.length;      // drafted token, negative: cached
            if (t >= 0 && (t >= a.tokens || !(mask[e >> 1] >> t & 1))) s[i][e] = -INFINITY;
          }
      }
      if (hidden) {
#pragma unroll 1
        for (int i = 0; i < kMine; ++i) {
          const int j = j0 + i;
          if (j >= seg.length || (unsigned)page_of(p, seg, j) < (unsigned)a.pages) continue;
#pragma unroll
          for (int k = 0; k < kMine / 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k * 8 + col + (e & 1) == i) s[k][e] = -INFINITY;
        }
      }

      // ---- running maximum and sum; weights in the values' type for the second product
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
        for (int i = 0; i < kMine / 8; ++i)
#pragma unroll
          for (int e = 2 * h; e < 2 * h + 2; ++e) {
            s[i][e] = exp2_approx(s[i][e] - base);
            total[h] += s[i][e];
          }
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= keep[e >> 1];

      // ---- infinities and NaN among the drafted values: a weight of zero must not meet them
      if (drafted) {
        const int from = max(seg.length - tile * kKeys, 0), upto = min(seg.length + a.tokens - tile * kKeys, kKeys);
        const uint32_t tile_values = smem_base + stage * 2 * kTileBytes + kTileBytes;
        bool odd = false;
        for (int i = tid; i < (upto - from) * kChunks; i += kThreads) {
          const int row = from + i / kChunks;
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(tile_values + row * kRowBytes + i % kChunks * 16) : "memory");
          odd = odd || is_odd<T>(w.x) || is_odd<T>(w.y) || is_odd<T>(w.z) || is_odd<T>(w.w);
        }
        if (__syncthreads_or(odd)) {
          // each is multiplied by the weights of the rows that see it only, and is zero in the product below
#pragma unroll 1
          for (int j = 0; j < kMine; ++j) {
            float w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float mine = 0.f;
#pragma unroll
              for (int k = 0; k < kMine / 8; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (k * 8 + e == (j & ~7) + (j & 1)) mine = s[k][2 * h + e];
              w[h] = __shfl_sync(0xffffffffu, mine, (lane & ~3) + (j & 7) / 2);
            }
            const int t = j0 + j - seg.length;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              uint32_t two;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two) : "r"(values + j * kRowBytes + ((i ^ (j & 7)) * 16) + col * 2) : "memory");
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t bits = e & 1 ? two >> 16 : two & 0xffffu;
                const bool sees = t >= 0 && t < a.tokens && (mask[e >> 1] >> t & 1);
                if (sees && (bits & Half16<T>::kExponent) == Half16<T>::kExponent) o[i][e] += w[e >> 1] * Half16<T>::value((uint16_t)bits);
              }
            }
          }
          __syncthreads();
          for (int i = tid; i < (upto - from) * D / 2; i += kThreads) {
            const uint32_t addr = tile_values + (from + i / (D / 2)) * kRowBytes + i % (D / 2) * 4;
            uint32_t two;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two) : "r"(addr) : "memory");
            constexpr uint32_t E = Half16<T>::kExponent;
            if ((two & E) == E) two &= 0xffff0000u;
            if ((two >> 16 & E) == E) two &= 0xffffu;
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(two) : "memory");
          }
          __syncthreads();
        }
      }

      // ---- weights times values
#pragma unroll
      for (int k = 0; k < kMine / 16; ++k) {
        const uint32_t w[4] = {Half16<T>::pack(s[2 * k][0], s[2 * k][1]), Half16<T>::pack(s[2 * k][2], s[2 * k][3]),
                               Half16<T>::pack(s[2 * k + 1][0], s[2 * k + 1][1]), Half16<T>::pack(s[2 * k + 1][2], s[2 * k + 1][3])};
        const int row = k * 16 + (lane & 15);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t v[4];
          ldsm_t(v, values + row * kRowBytes + (((2 * i + (lane >> 4)) ^ (row & 7)) * 16));
          Mma<T>::run(o[2 * i], w, v[0], v[1]);
          Mma<T>::run(o[2 * i + 1], w, v[2], v[3]);
        }
      }
      stage = (stage + 1) % kStages;

      put_place(page, turn);
    }

    // ---- the end of this CTA's keys for these rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      total[h] += __shfl_xor_sync(0xffffffffu, total[h], 1);
      total[h] += __shfl_xor_sync(0xffffffffu, total[h], 2);
    }
    if constexpr (kKeyWarps > 1) {
      // the warps that shared the keys pool their sums, the last one first
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
        const float mine = exp2_approx(top[h] - base);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][2 * h] *= mine;
          o[i][2 * h + 1] *= mine;
        }
        top[h] = m;
        total[h] = sum;
      }
      if (kKeyWarps == 4 && p.rows <= 4) {
        // there is room for the rows of all warps at once
        if (key_warp > 0 && quad < p.rows) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(pool + ((key_warp - 1) * 4 + quad) * D + i * 8 + col) = make_float2(o[i][0], o[i][1]);
        }
        __syncthreads();
        if (key_warp == 0 && quad < p.rows) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int w = 2; w >= 0; --w) {
              const float2 more = *reinterpret_cast<const float2*>(pool + (w * 4 + quad) * D + i * 8 + col);
              o[i][0] += more.x;
              o[i][1] += more.y;
            }
        }
        __syncthreads();
      } else {
#pragma unroll
        for (int part = 0; part < kRowWarps; ++part) {
#pragma unroll
          for (int w = kKeyWarps - 1; w >= 0; --w) {
            if (key_warp == w) {
#pragma unroll
              for (int i = 0; i < kPool / 8; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  float2* place = reinterpret_cast<float2*>(pool + (row_warp * 16 + quad + 8 * h) * kPool + i * 8 + col);
                  float (&mine)[4] = o[part * (kPool / 8) + i];
                  if (w < kKeyWarps - 1) {
                    const float2 sum = *place;
                    mine[2 * h] += sum.x;
                    mine[2 * h + 1] += sum.y;
                  }
                  if (w > 0) *place = make_float2(mine[2 * h], mine[2 * h + 1]);
                }
            }
            __syncthreads();
          }
        }
      }
    }
    const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
    auto out_row = [&](int r) {
      const int t = r / p.group, head = g * p.group + (r - t * p.group);
      return static_cast<T*>(a.out) + seg.b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2];
    };
    if (whole) {
      if (key_warp == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = row_warp * 16 + quad + 8 * h;
          if (r < p.rows) {
            // padding, and rows that see nothing, are zero
            const bool none = mask[h] == 0 || total[h] == 0.f;
            const float f = 1.f / total[h];
            T* out = out_row(r) + col;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
              *reinterpret_cast<uint32_t*>(out + 8 * i) = none ? 0u : Half16<T>::pack(o[i][2 * h] * f, o[i][2 * h + 1] * f);
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
          if (r < p.rows) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(slot + r * D + i * 8 + col) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
            if ((lane & 3) == 0) {
              slot[kRowTile * D + r] = top[h];
              slot[kRowTile * (D + 1) + r] = total[h];
            }
          }
        }
      }
      const int first_cta = seg.t0 == 0 ? cta : cta_of(units, ctas, seg.unit + p.overhead);
      const int last_cta = cta_of(units, ctas, seg.unit + p.overhead + seg.tiles - 1);
      const Joining join(first_cta, last_cta, cta, join_step(last_cta - first_cta + 1));
      // whether this CTA is the last of those that a counter waits for; what the others wrote is visible then
      auto last_at = [&](unsigned int* counter, int others) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const bool is_last = atomicAdd(counter, 1u) == (unsigned)others;
          if (is_last) *counter = 0;                               // for the next launch
          flags[1] = is_last;
        }
        __syncthreads();
        const bool is_last = flags[1] != 0;
        __threadfence();
        return is_last;
      };
      auto slot_of = [&](int c) { return p.partials + (size_t)(2 * c + (c == first_cta ? 1 : 0)) * kSlot; };
      // Joins `count` partials, `step` CTAs apart: into the output, or into the first one's slot.  A warp has two rows at a time, a lane four or two columns of
      // each; a lane fetches the maximum and total of one contributor, and eight contributors' sums are on their way together (one after the other took
      // a latency each; 24 rows of 19 contributors: 43 us in all then, 35 now).
      auto add_up = [&](int c0, int count, int step, bool ends) {
        constexpr int V = D / 32, kTogether = 8;
        for (int r0 = warp; r0 < p.rows; r0 += 8) {
          float m[2] = {-INFINITY, -INFINITY}, sum[2] = {}, acc[2][V] = {};
          const int rows[2] = {r0, r0 + 4 < p.rows ? r0 + 4 : r0};
          for (int k0 = 0; k0 < count; k0 += 32) {
            const int here = min(count - k0, 32);
            float by[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float* from = slot_of(c0 + (k0 + min(lane, here - 1)) * step) + kRowTile * D + rows[h];
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
                    v[e][h][i] = j0 + e < here ? __ldcg(reinterpret_cast<const float2*>(slot_of(c0 + (k0 + j0 + e) * step) + rows[h] * D + lane * V) + i) : make_float2(0.f, 0.f);
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
            if (r >= p.rows) break;
            if (ends) {
              const int t = r / p.group;
              const bool none = mask_of(p, seg.b, t) == 0 || sum[h] == 0.f;      // padding, and rows that see nothing, are zero
              const float f = 1.f / sum[h];
              T* out = out_row(r) + lane * V;
#pragma unroll
              for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(out + i) = none ? 0u : Half16<T>::pack(acc[h][i] * f, acc[h][i + 1] * f);
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
  }
  copies_wait<0>();
  if (tid == 0 && flags[0] && p.status) atomicExch(p.status, FP6M_ERR_BAD_ARG);
}

template <class T, int D, int kRowTile>
cudaError_t launch_tile(const TreeParams& p, int ctas, cudaStream_t stream) {
  constexpr int bytes = 3 * 128 / D * 2 * kKeys * D * 2 + 16 * D * 4 + 4 * 32 * 4 + sizeof(Plan) + 16 + 2 * kThreads * 8;
  cudaError_t e = allow_shared_memory<tree_attention_kernel<T, D, kRowTile>>(bytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(tree_attention_kernel<T, D, kRowTile>, dim3(ctas), dim3(kThreads), bytes, stream, p);
}
template <class T>
cudaError_t launch_tree(const TreeParams& p, int ctas, cudaStream_t stream) {
  if (p.a.head_dim == 64) return p.rows <= 16 ? launch_tile<T, 64, 16>(p, ctas, stream) : launch_tile<T, 64, 32>(p, ctas, stream);
  return p.rows <= 16 ? launch_tile<T, 128, 16>(p, ctas, stream) : launch_tile<T, 128, 32>(p, ctas, stream);
}

int tree_ctas(int sms) {
  const int want = sms > 0 ? 2 * sms : kMaxCtas;
  return want < kMaxCtas ? want : kMaxCtas;
}

// addresses and strides (in elements) of a tensor that is read or written sixteen bytes at a time
template <int kStrides>
bool rows_aligned(const void* p, const long long (&strides)[kStrides]) {
  bool ok = p && aligned16(p);
  for (long long s : strides) ok = ok && s >= 0 && s % 8 == 0;
  return ok;
}

}  // namespace

extern "C" {

size_t fp6m_tree_attention_scratch_bytes(int sms) {
  const size_t few = (size_t)tree_ctas(sms) * 2 * kFewRows * (128 + 2) * sizeof(float), many = tree_tc5_partial_bytes(sms);
  return kCounterBytes + (few > many ? few : many);
}

int fp6m_tree_attention(const fp6m_tree_attention_args* args, void* scratch, size_t scratch_bytes, int dev, void* stream, int* status_dev) {
  if (!args) return FP6M_ERR_BAD_ARG;
  const fp6m_tree_attention_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.heads < 0 || (a.type != FP6M_TYPE_F16 && a.type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (a.tokens > 64 || (a.head_dim != 64 && a.head_dim != 128)) return FP6M_ERR_PROB_SHAPE;
  if (a.batch == 0 || a.tokens == 0 || a.heads == 0) return FP6M_OK;
  if (a.kv_heads <= 0 || a.heads % a.kv_heads) return FP6M_ERR_PROB_SHAPE;
  // (pages are looked up in blocks of up to 2048 tokens, two of them ahead, so tokens stay that far from 2^31)
  if (a.max_pages < 0 || a.pages < 0 || a.page_size <= 0 || (long long)a.max_pages * a.page_size > 0x7fff0000ll) return FP6M_ERR_PROB_SHAPE;
  if ((long long)a.tokens * a.heads > 0xffffffll) return FP6M_ERR_PROB_SHAPE;
  if (!rows_aligned(a.q, a.q_stride) || !rows_aligned(a.k, a.k_stride) || !rows_aligned(a.v, a.v_stride) || !rows_aligned(a.out, a.out_stride)) return FP6M_ERR_BAD_ARG;
  if (!a.lengths || !a.tree || a.tree_stride < 0 || !scratch || !aligned16(scratch)) return FP6M_ERR_BAD_ARG;
  if (a.max_pages > 0 && (!rows_aligned(a.k_cache, a.k_cache_stride) || !rows_aligned(a.v_cache, a.v_cache_stride) || !a.page_table || a.page_table_stride < 0)) return FP6M_ERR_BAD_ARG;
  DeviceGuard guard(dev);
  const int sms = sm_count(dev);
  if (sms <= 0) return cuda_fail(cudaGetLastError(), "cudaDeviceGetAttribute");
  if (scratch_bytes < fp6m_tree_attention_scratch_bytes(sms)) return FP6M_ERR_SCRATCH;
  TreeParams p;
  p.a = a;
  p.group = a.heads / a.kv_heads;
  p.rows = a.tokens * p.group;
  p.row_tiles = p.parts = 1;
  p.overhead = 4;
  int log2 = 0;
  while ((1ll << log2) < a.page_size) ++log2;
  p.page_shift = 31 + log2;
  p.page_magic = ((1ull << p.page_shift) + a.page_size - 1) / a.page_size;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  if (p.scale_log2 == 0.f) p.scale_log2 = 1e-37f;      // a masked score of minus infinity stays that
  p.arrived = static_cast<unsigned int*>(scratch);
  p.partials = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + kCounterBytes);
  p.status = status_dev;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p.rows > kFewRows ? launch_tree_tc5(p, sms, st)
                        : a.type == FP6M_TYPE_F16 ? launch_tree<half>(p, tree_ctas(sms), st) : launch_tree<__nv_bfloat16>(p, tree_ctas(sms), st);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "tree_attention launch");
}

}  // extern "C"
