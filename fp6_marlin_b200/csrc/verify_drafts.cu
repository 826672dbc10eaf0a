// Which drafted tokens are accepted, and the token after them (include/fp6m.h: fp6m_verify_drafts).
//
//   a child c of the last accepted token n is accepted where u_c q(c) < r(c), else r <- max(r - q, 0) / sum;   r = p = target[n] at first, q = draft[n]
//   none accepted: the next token is the lowest x with sum_{y <= x} r(y) > u_0 sum r
//
// However often r is reduced, it stays r = max(alpha p - beta q, 0): max(max(a, 0) / Z - q, 0) = max(a / Z - q, 0) for q >= 0, so a reduction by q changes beta to
// beta + 1 and the division by its sum Z both to alpha / Z and beta / Z.  Two numbers are all that is kept, and the rows of p and q are read only where a sum is
// needed: for a second child of a token whose first was not accepted, and for the next token.  Without draft r is alpha p, with zeros at the children that were
// not accepted.
//
// Sums are taken in 64 bits: neighbouring sums of a row of 10^5 probabilities lie 10^-5 apart, and sums in 32 bits, off by 10^-7, would choose another token once in a hundred times.
//
// A cluster of CTAs a sequence: every warp sums a stretch of the row, the sums are exchanged through distributed shared memory, and every CTA goes the same way
// through the tree.  What decides about a token - its probabilities in its parent's rows and its random number - is fetched for all tokens at once, before.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>

#include "../../include/fp6m.h"
#include "device_utils.cuh"
#include "host_common.h"

namespace {

using namespace fp6m;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostTokens = 64, kMostCluster = 8;

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

// r = max(alpha p - beta q, 0), or alpha p with holes
template <class P>
struct Rest {
  const P *p, *q;                        // q null: no draft
  double alpha, beta;
  const int* holes;                      // ids whose probability is gone (no draft)
  int hole_count;
  __device__ __forceinline__ double of(float p_value, float q_value) const {
    const double x = alpha * (double)clean(p_value);
    return q ? fmax(fma(-beta, (double)clean(q_value), x), 0.0) : x;
  }
  __device__ __forceinline__ bool hole(int x) const {
    for (int i = 0; i < hole_count; ++i)
      if (holes[i] == x) return true;
    return false;
  }
};

// Calls take(first id, values[N]) for the warp's lanes with N neighbouring values of r each, from..upto in steps of 32 N.  `from` is a multiple of 32 N from `start`, which is
// minus the number of values by which the rows lie behind a 16-byte boundary; a step that is not wholly inside the row comes by single values.
template <class P, class Take>
__device__ __forceinline__ void for_values(const Rest<P>& r, int vocab, int start, bool vectors, bool any_holes, int from, int upto, Take&& take) {
  constexpr int N = 16 / sizeof(P), kStep = 32 * N, kTogether = 4;
  const int lane = threadIdx.x & 31;
  for (int base = from; base < upto; base += kStep * kTogether) {
    uint4 pv[kTogether], qv[kTogether];
    bool whole[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int first = start + base + k * kStep;
      whole[k] = vectors && base + k * kStep < upto && first >= 0 && first + kStep <= vocab;
      const uint4 none = make_uint4(0, 0, 0, 0);
      pv[k] = whole[k] ? __ldg(reinterpret_cast<const uint4*>(r.p + first) + lane) : none;
      qv[k] = whole[k] && r.q ? __ldg(reinterpret_cast<const uint4*>(r.q + first) + lane) : none;
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      if (base + k * kStep >= upto) return;
      const int x = start + base + k * kStep + lane * N;
      float pf[N], qf[N];
      Probability<P>::unpack(pv[k], pf);
      Probability<P>::unpack(qv[k], qf);
      if (!whole[k]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool there = x + i >= 0 && x + i < vocab;
          pf[i] = there ? Probability<P>::value(r.p + x + i) : 0.f;
          qf[i] = there && r.q ? Probability<P>::value(r.q + x + i) : 0.f;
        }
      }
      double v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = r.of(pf[i], qf[i]);
      if (any_holes) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (r.hole(x + i)) v[i] = 0.0;
      }
      if (!take(x, v)) return;
    }
  }
}

template <class P>
__global__ void __launch_bounds__(kThreads) verify_drafts_kernel(const __grid_constant__ fp6m_verify_drafts_args a) {
  constexpr int N = 16 / sizeof(P), kStep = 32 * N;
  __shared__ double sums[2][kWarps];                                // of the warps' stretches, in turn
  __shared__ float p_of[kMostTokens], q_of[kMostTokens], u_of[kMostTokens];
  __shared__ int parent[kMostTokens], id_of[kMostTokens], holes[kMostTokens];
  __shared__ unsigned long long masks[kMostTokens];
  __shared__ double every[kMostCluster * kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int b = blockIdx.x / ranks;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const P* target = static_cast<const P*>(a.target) + b * a.target_stride[0];
  const P* draft = a.draft ? static_cast<const P*>(a.draft) + b * a.draft_stride[0] : nullptr;
  // ---- all that the way through the tree depends on
  if (tid < a.tokens) {
    const unsigned long long mask = a.tree[b * a.tree_stride + tid], earlier = mask & ((1ull << tid) - 1);
    const int above = mask ? 63 - __clzll(earlier) : -2;             // the last earlier token that it sees, -1: none; -2: padding
    const long long id = a.drafted[(long long)b * a.tokens + tid];
    const bool inside = id >= 0 && id < a.vocab && above >= 0;
    masks[tid] = mask;
    parent[tid] = above;
    id_of[tid] = inside ? (int)id : -1;
    p_of[tid] = inside ? clean(Probability<P>::value(target + above * a.target_stride[1] + id)) : 0.f;
    q_of[tid] = inside ? (draft ? clean(Probability<P>::value(draft + above * a.draft_stride[1] + id)) : 1.f) : 0.f;
    u_of[tid] = a.uniforms[(long long)b * a.tokens + tid];
  }
  __syncthreads();
  const bool alive = masks[0] != 0;                                  // (the same in all CTAs of the cluster)

  Rest<P> r = {target, draft, 1.0, 0.0, holes, 0};
  int node = 0, count = alive ? 1 : 0, start = 0, stretch = 0, pass = 0;
  bool vectors = false;
  double whole = 0.0;
  // The sum of r, and in `every` those of the stretches of all warps of the cluster, in their order.
  auto add_up = [&] {
    const uintptr_t off = reinterpret_cast<uintptr_t>(r.p) & 15;
    vectors = off % sizeof(P) == 0 && (!r.q || (reinterpret_cast<uintptr_t>(r.q) & 15) == off);
    start = vectors ? -(int)(off / sizeof(P)) : 0;
    const int steps = (a.vocab - start + kStep - 1) / kStep, workers = ranks * kWarps;
    stretch = (steps + workers - 1) / workers * kStep;
    const int me = rank * kWarps + warp;
    const long long from = (long long)me * stretch;
    const int end = a.vocab - start;
    double sum = 0.0;
    if (from < end) {
      const int upto = (int)min(from + stretch, (long long)end);
      bool any_holes = false;
      for (int i = 0; i < r.hole_count; ++i) any_holes = any_holes || (holes[i] >= start + from && holes[i] < start + upto);
      for_values(r, a.vocab, start, vectors, any_holes, (int)from, upto, [&](int, double (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) sum += v[i];
        return true;
      });
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[pass & 1][warp] = sum;
    cluster_sync();
    for (int i = tid; i < workers; i += kThreads) every[i] = remote_double(smem_u32(&sums[pass & 1][i % kWarps]), i / kWarps);
    ++pass;
    __syncthreads();
    whole = 0.0;
    for (int i = lane; i < workers; i += 32) whole += every[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) whole += __shfl_xor_sync(0xffffffffu, whole, o);
  };
  auto go_to = [&](int n) {
    node = n;
    r.p = target + n * a.target_stride[1];
    r.q = nullptr;                                                   // nothing to subtract yet
    r.alpha = 1.0;
    r.beta = 0.0;
    r.hole_count = 0;
  };

  // ---- the way through the tree
  bool reduced = false, gone = false;                                // r has been reduced since its sum was taken; nothing of it remains
  go_to(0);
  for (int i = 1; alive && i < a.tokens; ++i) {
    if (parent[i] != node) continue;
    if (reduced) {
      // a further child: r is divided by its sum
      add_up();
      gone = !(whole > 0.0);
      if (!gone) {
        r.alpha /= whole;
        r.beta /= whole;
      }
      reduced = false;
    }
    bool is_hole = false;
    for (int k = 0; k < r.hole_count; ++k) is_hole = is_hole || (holes[k] == id_of[i] && id_of[i] >= 0);
    const double mine = gone || is_hole ? 0.0 : fmax(fma(-r.beta, (double)q_of[i], r.alpha * (double)p_of[i]), 0.0);
    const double left = draft ? mine : gone || is_hole ? 0.0 : r.alpha * (double)p_of[i];
    if ((double)u_of[i] * (double)q_of[i] < left) {
      if (rank == 0 && tid == 0) a.accepted[(long long)b * a.tokens + count] = i;
      ++count;
      go_to(i);
      gone = false;
    } else {
      if (draft) {
        r.q = draft + node * a.draft_stride[1];
        r.beta += 1.0;
      } else if (id_of[i] >= 0 && !is_hole) {
        __syncthreads();
        if (tid == 0) holes[r.hole_count] = id_of[i];
        __syncthreads();
        ++r.hole_count;
      }
      reduced = !gone;
    }
  }

  // ---- the next token
  long long next = -1;
  if (alive) {
    if (!gone) add_up();
    if (gone || !(whole > 0.0)) {
      go_to(node);
      add_up();
    }
  }
  const bool any = alive && whole > 0.0;
  int owner = -1;
  double before = 0.0;
  const double goal = (double)u_of[0] * whole;
  if (any) {
    // the first stretch with which the sum exceeds the goal; where rounding leaves none, the last that holds something
    const int workers = ranks * kWarps;
    double upto = 0.0;
    for (int i0 = 0; i0 < workers && owner < 0; i0 += 32) {
      const double x = i0 + lane < workers ? every[i0 + lane] : 0.0;
      double sum = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
      }
      sum += upto;
      const unsigned over = __ballot_sync(0xffffffffu, sum > goal && x > 0.0);
      if (over) {
        owner = i0 + __ffs(over) - 1;
        before = __shfl_sync(0xffffffffu, sum - x, __ffs(over) - 1);
      }
      upto = __shfl_sync(0xffffffffu, sum, 31);
    }
    if (owner < 0) {
      for (int i0 = 0; i0 < workers; i0 += 32) {
        const unsigned some = __ballot_sync(0xffffffffu, i0 + lane < workers && every[i0 + lane] > 0.0);
        if (some) owner = i0 + 31 - __clz(some);
      }
      before = -INFINITY;                                            // no sum exceeds the goal
    }
  }
  if (any && owner == rank * kWarps + warp) {
    const long long from = (long long)owner * stretch;
    const int end = a.vocab - start, upto = (int)min(from + stretch, (long long)end);
    bool any_holes = false;
    for (int i = 0; i < r.hole_count; ++i) any_holes = any_holes || (holes[i] >= start + from && holes[i] < start + upto);
    double sum = before;
    int found = -1, last = -1;
    for_values(r, a.vocab, start, vectors, any_holes, (int)from, upto, [&](int x, double (&v)[N]) {
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
      const double below = sum + (incl - mine);
      int here = -1;
      double at = below;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        at += v[i];
        if (here < 0 && v[i] > 0.0 && at > goal) here = x + i;
      }
      const unsigned over = __ballot_sync(0xffffffffu, here >= 0);
      const unsigned some = __ballot_sync(0xffffffffu, mine_last >= 0);
      if (some) last = __shfl_sync(0xffffffffu, mine_last, 31 - __clz(some));
      if (over) {
        found = __shfl_sync(0xffffffffu, here, __ffs(over) - 1);
        return false;
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
      return true;
    });
    next = found >= 0 ? found : last;
    if (lane == 0) a.next_tokens[b] = next;
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

template <class P>
cudaError_t launch(const fp6m_verify_drafts_args& a, int ranks, cudaStream_t stream) {
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
  const int ranks = kMostCluster;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.type == FP6M_TYPE_F32 ? launch<float>(a, ranks, st) : a.type == FP6M_TYPE_F16 ? launch<half>(a, ranks, st) : launch<__nv_bfloat16>(a, ranks, st);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "verify_drafts launch");
}
