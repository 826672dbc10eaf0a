// Which drafted tokens are accepted, and the token after them (include/fp6m.h: fp6m_verify_drafts).
//
//   a child c of the last accepted token n is accepted where u_c q(c) < r(c), else r <- max(r - q, 0) / sum;   r = p = target[n] at first, q = draft[n]
//   none accepted: the next token is the lowest x with sum_{y <= x} r(y) > u_0 sum r
//
// However often r is reduced, it stays r = max(p - q - less q, 0) / S: with less = 0 after the first reduction by q, and with S the sum of the numerators, a division by the sum makes S of 1,
// and max(max(a, 0) / S - q, 0) = max(a - S q, 0) / S for q >= 0, so a further reduction adds S to `less`.  Two numbers are all that is kept, and the rows of p and q are read only
// where a sum is needed: for a second child of a token whose first was not accepted, and for the next token.  (p - q first: 64 bits hold the difference of neighbours, so nothing is left where p = q, and
// no error of p is left where p - q is small; in alpha p - beta q both were.)  Without draft r is p / S, with zeros at the children that were not
// accepted, and one sum, of p without any of the children, serves all of a token's children: what they have is added to it.
//
// Sums are taken in 64 bits: neighbouring sums of a row of 10^5 probabilities lie 10^-5 apart, and sums in 32 bits, off by 10^-7, would choose another token once in a hundred times.
//
// A cluster of CTAs a sequence: every warp sums a stretch of the row, chunk by chunk, the sums are exchanged through distributed shared memory, every CTA goes the same way
// through the tree, and in the end one warp looks through the one chunk that the drawn number falls into.  What decides about a token - its probabilities in its parent's rows and
// its random number - is fetched for all tokens at once, before.
//
// Bound by latencies that follow one another: launch and the tokens' numbers (about 4 us), then for each sum a round of loads, an exchange and a decision (about 2 us), and the search (1.5 us).  One
// sequence, vocabulary 32000, no draft: 7.0 us; five trees of sixteen tokens, 50257: 20.4; 64 chains of seven, 131072, 32 bits: 20.3, where its one sum a sequence reads 3.3 TB/s over the whole call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/fp6m.h"
#include "device_utils.cuh"
#include "host_common.h"

namespace {

using namespace fp6m;

constexpr int kThreads = 256, kWarps = kThreads / 32, kCtas = 3;      // per multiprocessor
constexpr int kMostTokens = 64, kPortable = 8, kMostCluster = 16, kChunks = 32;       // chunks of a stretch at most

template <class P> struct Probability;
template <> struct Probability<float> {
  static __device__ __forceinline__ float value(const float* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) { f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w); }
};
template <> struct Probability<half> {
  static __device__ __forceinline__ float value(const half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 two = __half22float2(*reinterpret_cast<const half2*>(&w[i]));
      f[2 * i] = two.x;
      f[2 * i + 1] = two.y;
    }
  }
};
template <> struct Probability<__nv_bfloat16> {
  static __device__ __forceinline__ float value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
// what is negative, infinite or NaN counts as nothing
__device__ __forceinline__ float clean(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double remote_double(uint32_t addr, int rank) {
  uint32_t there;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(there) : "memory");
  return v;
}

// The numerator of r: max(p - q - less q, 0), or p with holes
template <class P>
struct Rest {
  const P *p, *q;                        // q null: nothing is subtracted
  double less;
  const int* holes;                      // ids whose probability is gone (no draft)
  int hole_count;
  __device__ __forceinline__ double of(float p_value, float q_value) const {
    const double p_clean = clean(p_value), q_clean = clean(q_value);
    return q ? fmax(fma(-less, q_clean, p_clean - q_clean), 0.0) : p_clean;
  }
  __device__ __forceinline__ bool hole(int x) const {
    for (int i = 0; i < hole_count; ++i)
      if (holes[i] == x) return true;
    return false;
  }
};

// Calls take(first id, values[N]) for the warp's lanes with N neighbouring values of r each, from..upto in groups of kTogether steps of 32 N.  `from` is a multiple of a group from
// `start`, which is minus the number of values by which the rows lie behind a 16-byte boundary.  Groups that are wholly inside the row come by vectors, and there only negative values
// and NaN are looked for: `odd` says that infinities of q were met (those of p show in the sum).  Other groups come by single values.
constexpr int kTogether = 4;             // steps whose loads are on their way together
template <class P, class Take>
__device__ __forceinline__ void for_values(const Rest<P>& r, int vocab, int start, bool vectors, bool any_holes, int from, int upto, bool& odd, Take&& take) {
  constexpr int N = 16 / sizeof(P), kStep = 32 * N;
  const int lane = threadIdx.x & 31;
  const double minus_less = -r.less;
  auto vector_group = [&](int first, auto subtracts) {
    constexpr bool kSubtracts = decltype(subtracts)::value;
    uint4 pv[kTogether], qv[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      pv[k] = __ldg(reinterpret_cast<const uint4*>(r.p + first + k * kStep) + lane);
      if (kSubtracts) qv[k] = __ldg(reinterpret_cast<const uint4*>(r.q + first + k * kStep) + lane);
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      float pf[N], qf[N];
      double v[N];
      Probability<P>::unpack(pv[k], pf);
      if (kSubtracts) Probability<P>::unpack(qv[k], qf);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float p = fmaxf(pf[i], 0.f);
        if (kSubtracts) {
          const float q = fmaxf(qf[i], 0.f);
          odd = odd || q == INFINITY;
          const double x = fma(minus_less, (double)q, (double)p - (double)q);
          v[i] = __double2hiint(x) < 0 ? 0.0 : x;
        } else {
          v[i] = (double)p;
        }
      }
      const int x = first + k * kStep + lane * N;
      if (any_holes) {
        for (int h = 0; h < r.hole_count; ++h) {
          const int at = r.holes[h] - x;
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (at == i) v[i] = 0.0;
        }
      }
      if (!take(x, v)) return false;
    }
    return true;
  };
#pragma unroll 1
  for (int base = from; base < upto; base += kStep * kTogether) {
    const int first = start + base;
    if (vectors && first >= 0 && first + kStep * kTogether <= vocab) {
      if (!(r.q ? vector_group(first, std::true_type()) : vector_group(first, std::false_type()))) return;
    } else {
#pragma unroll 1
      for (int k = 0; k < kTogether; ++k) {
        const int x = first + k * kStep + lane * N;
        double v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool there = x + i >= 0 && x + i < vocab;
          v[i] = there ? r.of(Probability<P>::value(r.p + x + i), r.q ? Probability<P>::value(r.q + x + i) : 0.f) : 0.0;
          if (any_holes && r.hole(x + i)) v[i] = 0.0;
        }
        if (!take(x, v)) return;
      }
    }
  }
}

// the sum over the lanes, in all of them
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The first of n numbers with which their sum exceeds the goal, and the sum before it; where none does, the last that is not zero, and minus infinity.  Called by a warp.
__device__ __forceinline__ int find_first(const double* numbers, int n, double goal, double before, double& sum_before) {
  const int lane = threadIdx.x & 31;
  int last = -1;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const double x = i0 + lane < n ? numbers[i0 + lane] : 0.0;
    double sum = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double other = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += other;
    }
    sum += before;
    const unsigned over = __ballot_sync(0xffffffffu, sum > goal && x > 0.0), some = __ballot_sync(0xffffffffu, x > 0.0);
    if (over) {
      sum_before = __shfl_sync(0xffffffffu, sum - x, __ffs(over) - 1);
      return i0 + __ffs(over) - 1;
    }
    if (some) last = i0 + 31 - __clz(some);
    before = __shfl_sync(0xffffffffu, sum, 31);
  }
  sum_before = -INFINITY;
  return last;
}

template <class P>
__global__ void __launch_bounds__(kThreads, kCtas) verify_drafts_kernel(const __grid_constant__ fp6m_verify_drafts_args a) {
  constexpr int N = 16 / sizeof(P), kStep = 32 * N;
  __shared__ double sums[2][kWarps];                                // of the warps' stretches, in turn
  __shared__ double fine[kWarps][kChunks];                          // of a stretch's chunks
  __shared__ double every[kMostCluster * kWarps];
  __shared__ float p_of[kMostTokens], q_of[kMostTokens], u_of[kMostTokens];
  __shared__ int parent[kMostTokens], id_of[kMostTokens], holes[kMostTokens];
  __shared__ unsigned long long children[kMostTokens], firsts;      // of a token; those whose id is in the vocabulary and that of no sister before them
  __shared__ bool lives;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int b = blockIdx.x / ranks, workers = ranks * kWarps;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < kMostTokens) children[tid] = 0;
  if (tid == 0) firsts = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const P* target = static_cast<const P*>(a.target) + b * a.target_stride[0];
  const P* draft = a.draft ? static_cast<const P*>(a.draft) + b * a.draft_stride[0] : nullptr;
  // ---- all that the way through the tree depends on
  if (tid < a.tokens) {
    const unsigned long long mask = a.tree[b * a.tree_stride + tid], earlier = mask & ((1ull << tid) - 1);
    const int above = mask ? 63 - __clzll(earlier) : -2;             // the last earlier token that it sees, -1: none; -2: padding
    const long long id = a.drafted[(long long)b * a.tokens + tid];
    const bool inside = id >= 0 && id < a.vocab && above >= 0;
    if (tid == 0) lives = mask != 0;
    if (above >= 0) atomicOr(&children[above], 1ull << tid);         // (the result does not depend on the order)
    parent[tid] = above;
    id_of[tid] = inside ? (int)id : -1;
    p_of[tid] = inside ? clean(Probability<P>::value(target + above * a.target_stride[1] + id)) : 0.f;
    q_of[tid] = inside ? (draft ? clean(Probability<P>::value(draft + above * a.draft_stride[1] + id)) : 1.f) : 0.f;
    u_of[tid] = a.uniforms[(long long)b * a.tokens + tid];
  }
  __syncthreads();
  if (!draft && a.tokens > 1) {
    if (tid < a.tokens && id_of[tid] >= 0) {
      bool first = true;
      for (int k = parent[tid] + 1; k < tid; ++k) first = first && (parent[k] != parent[tid] || id_of[k] != id_of[tid]);
      if (first) atomicOr(&firsts, 1ull << tid);
    }
    __syncthreads();
  }
  const bool alive = lives;                                          // (the same in all CTAs of the cluster)

  Rest<P> r = {target, nullptr, 0.0, holes, 0};
  double over = 1.0;                     // S
  int node = 0, count = alive ? 1 : 0, start = 0, stretch = 0, chunk = 0, pass = 0;
  bool vectors = false;
  double whole = 0.0;
  auto has_holes = [&](long long from, long long upto) {
    bool any = false;
    for (int i = 0; i < r.hole_count; ++i) any = any || (holes[i] >= start + from && holes[i] < start + upto);
    return any;
  };
  // The sum of r; in `every` those of the stretches of all warps of the cluster, in `fine` those of this warp's chunks, in their order.
  auto add_up = [&] {
    const uintptr_t off = reinterpret_cast<uintptr_t>(r.p) & 15;
    vectors = off % sizeof(P) == 0 && (!r.q || (reinterpret_cast<uintptr_t>(r.q) & 15) == off);
    start = vectors ? -(int)(off / sizeof(P)) : 0;
    const int end = a.vocab - start, steps = (end + kStep - 1) / kStep;
    const int groups = ((steps + workers - 1) / workers + kTogether - 1) / kTogether;      // of a stretch
    stretch = groups * kTogether * kStep;
    chunk = (groups + kChunks - 1) / kChunks * kTogether * kStep;
    bool again = false;
#pragma unroll 1
    while (true) {
      const long long from = (long long)(rank * kWarps + warp) * stretch;
      double sum = 0.0;
      bool odd = false;
      if (from < end) {
        const int upto = (int)min(from + stretch, (long long)end);
        const bool any_holes = has_holes(from, upto);
#pragma unroll 1
        for (int c = 0; from + (long long)c * chunk < upto; ++c) {
          double part = 0.0;
          for_values(r, a.vocab, start, vectors, any_holes, (int)from + c * chunk, min((int)min(from + (long long)(c + 1) * chunk, (long long)end), upto), odd, [&](int, double (&v)[N]) {
            double two[2] = {};
#pragma unroll
            for (int i = 0; i < N; ++i) two[i & 1] += v[i];
            part += two[0] + two[1];
            return true;
          });
          part = warp_sum(part);
          if (lane == 0) fine[warp][c] = part;
          sum += part;
        }
      }
      if (__any_sync(0xffffffffu, odd)) sum = __longlong_as_double(0x7ff8000000000000ll);
      if (lane == 0) sums[pass & 1][warp] = sum;
      cluster_sync();
      for (int i = tid; i < workers; i += kThreads) every[i] = remote_double(smem_u32(&sums[pass & 1][i % kWarps]), i / kWarps);
      ++pass;
      __syncthreads();
      whole = 0.0;
      for (int i = lane; i < workers; i += 32) whole += every[i];
      whole = warp_sum(whole);
      if (again || (__double2hiint(whole) & 0x7ff00000) != 0x7ff00000) break;
      again = true;                                                  // there are infinities: value by value
      vectors = false;
    }
  };
  auto go_to = [&](int n) {
    node = n;
    r.p = target + n * a.target_stride[1];
    r.q = nullptr;                                                   // nothing to subtract yet
    r.less = 0.0;
    r.hole_count = 0;
    over = 1.0;
  };

  // ---- the way through the tree.  (The sums are taken in one place, so that the code is there once.)
  bool reduced = false, gone = false;      // r has been reduced and not been divided by its sum since; nothing of it remains
  bool summed = false, last_sum = false;   // `whole` is the sum of r, without draft that of the row without the children; it is that of the row itself
  go_to(0);
  unsigned long long rest = children[0];   // of the node, those that have not had their turn
#pragma unroll 1
  while (alive) {
    bool asks = false;                     // a further child asks for the sum
    while (rest && !last_sum) {
      const int i = __ffsll(rest) - 1;
      if (reduced) {
        if (!summed) {
          asks = true;
          break;
        }
        double left = whole;
        if (!draft) {                      // the children that are still to come
          const unsigned long long of = rest & firsts;
          left += warp_sum((of >> lane & 1 ? (double)p_of[lane] : 0.0) + (of >> (lane + 32) & 1 ? (double)p_of[lane + 32] : 0.0));
        }
        gone = !(left > 0.0);
        if (!gone) over = left;
        reduced = false;
        if (draft) summed = false;
      }
      const bool nothing = gone || (!draft && !(firsts >> i & 1));   // an id that was not accepted before has nothing left
      if (!nothing && (double)u_of[i] * (double)q_of[i] * over < r.of(p_of[i], q_of[i])) {
        if (rank == 0 && tid == 0) a.accepted[(long long)b * a.tokens + count] = i;
        ++count;
        go_to(i);
        rest = children[i];
        gone = summed = reduced = false;
      } else {
        rest &= rest - 1;
        if (draft) {
          if (r.q) r.less += over;
          r.q = draft + node * a.draft_stride[1];
        }
        reduced = !gone;
      }
    }
    // ---- the next token is drawn from r, without draft from the row without the children (none has been accepted); from the row itself if that is nothing
    if (!asks) {
      if (summed && (whole > 0.0 || last_sum)) break;
      if (summed || (draft && gone)) {
        go_to(node);
        last_sum = true;
      }
    }
    if (!draft && !last_sum) {
      const unsigned long long of = children[node] & firsts;
      if (of) {
        __syncthreads();
        if (tid < kMostTokens && of >> tid & 1) holes[__popcll(of & ((1ull << tid) - 1))] = id_of[tid];
        __syncthreads();
      }
      r.hole_count = __popcll(of);
    }
    add_up();
    summed = true;
  }
  const bool any = alive && whole > 0.0;
  if (any) {
    const double goal = (double)u_of[0] * whole;
    double before;
    const int owner = find_first(every, workers, goal, 0.0, before);
    if (owner == rank * kWarps + warp) {
      // this warp's stretch; in it the chunk, in that the token
      __syncwarp();
      const long long from = (long long)owner * stretch;
      const int end = a.vocab - start, upto = (int)min(from + stretch, (long long)end), chunks = (int)((upto - from + chunk - 1) / chunk);
      const int c = find_first(fine[warp], chunks, goal, before, before);
      const int first = (int)from + c * chunk, behind = (int)min((long long)first + chunk, (long long)upto);
      double sum = before;
      int found = -1, last = -1;
      bool odd = false;
      for_values(r, a.vocab, start, vectors, has_holes(first, behind), first, behind, odd, [&](int x, double (&v)[N]) {
        double mine = 0.0;
        int mine_last = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          mine += v[i];
          if (v[i] > 0.0) mine_last = x + i;
        }
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double other = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += other;
        }
        int here = -1;
        double at = sum + (incl - mine);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          at += v[i];
          if (here < 0 && v[i] > 0.0 && at > goal) here = x + i;
        }
        const unsigned over = __ballot_sync(0xffffffffu, here >= 0), some = __ballot_sync(0xffffffffu, mine_last >= 0);
        if (some) last = __shfl_sync(0xffffffffu, mine_last, 31 - __clz(some));
        if (over) {
          found = __shfl_sync(0xffffffffu, here, __ffs(over) - 1);
          return false;
        }
        sum += __shfl_sync(0xffffffffu, incl, 31);
        return true;
      });
      if (lane == 0) a.next_tokens[b] = found >= 0 ? found : last;
    }
  }
  if (rank == 0) {
    if (tid == 0) {
      a.counts[b] = count;
      if (alive) a.accepted[(long long)b * a.tokens] = 0;
      if (!any) a.next_tokens[b] = -1;
    }
    if (tid >= count && tid < a.tokens) a.accepted[(long long)b * a.tokens + tid] = -1;
  }
  cluster_sync();                                                    // (the others may still read this CTA's sums)
}

// The most CTAs that a cluster of this kernel may have on a device: more than eight have to be allowed, and a part of a GPU may have room for fewer.  Asked once for each device.
template <class P>
cudaError_t largest_cluster(int dev, int* most) {
  static std::atomic<int> known[64];
  if (dev < 64 && (*most = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(verify_drafts_kernel<P>), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kMostCluster);
  cfg.blockDim = dim3(kThreads);
  e = cudaOccupancyMaxPotentialClusterSize(most, verify_drafts_kernel<P>, &cfg);
  if (e != cudaSuccess) return e;
  if (*most < 1) *most = 1;
  if (dev < 64) known[dev].store(*most, std::memory_order_relaxed);
  return cudaSuccess;
}

template <class P>
cudaError_t launch(const fp6m_verify_drafts_args& a, int dev, int ranks, cudaStream_t stream) {
  int most = 0;
  const cudaError_t e = largest_cluster<P>(dev, &most);
  if (e != cudaSuccess) return e;
  ranks = std::min(ranks, most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)ranks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_drafts_kernel<P>, a);
}

}  // namespace

extern "C" int fp6m_verify_drafts(const fp6m_verify_drafts_args* args, int dev, void* stream) {
  if (!args) return FP6M_ERR_BAD_ARG;
  const fp6m_verify_drafts_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.vocab < 0 || (a.type != FP6M_TYPE_F32 && a.type != FP6M_TYPE_F16 && a.type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (a.tokens > kMostTokens || a.vocab > 1 << 30 || a.batch > INT_MAX / kMostCluster) return FP6M_ERR_PROB_SHAPE;
  if (a.batch == 0 || a.tokens == 0) return FP6M_OK;
  if (a.vocab == 0) return FP6M_ERR_PROB_SHAPE;
  const uintptr_t size = a.type == FP6M_TYPE_F32 ? 4 : 2;
  if (!a.target || !a.drafted || !a.tree || !a.uniforms || !a.accepted || !a.counts || !a.next_tokens || reinterpret_cast<uintptr_t>(a.target) % size ||
      reinterpret_cast<uintptr_t>(a.draft) % size || a.tree_stride < 0)
    return FP6M_ERR_BAD_ARG;
  for (int i = 0; i < 2; ++i)
    if (a.target_stride[i] < 0 || (a.draft && a.draft_stride[i] < 0)) return FP6M_ERR_BAD_ARG;
  DeviceGuard guard(dev);
  const int sms = sm_count(dev);
  if (sms <= 0) return cuda_fail(cudaGetLastError(), "cudaDeviceGetAttribute");
  // As many CTAs a sequence as run at once, and as have a group of steps for every warp.  More than eight must share a group of multiprocessors that not all groups have room for, so only where
  // two per multiprocessor are enough: 8 / 16 at most, eight tokens over 128000: one sequence 11.3 / 9.6 us, 16 sequences 14.9 / 13.2, but 27 (four tokens) 15.0 / 20.9, 40 15.9 / 24.2.
  const long long group = kTogether * 32 * (16 / (int)size), fit = (long long)kCtas * sms / a.batch, useful = (a.vocab + group * kWarps - 1) / (group * kWarps);
  const long long most = (long long)a.batch * kMostCluster <= 2ll * sms ? kMostCluster : kPortable;
  const int ranks = (int)std::max(1ll, std::min({fit, useful, most}));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.type == FP6M_TYPE_F32 ? launch<float>(a, dev, ranks, st) : a.type == FP6M_TYPE_F16 ? launch<half>(a, dev, ranks, st) : launch<__nv_bfloat16>(a, dev, ranks, st);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "verify_drafts launch");
}
