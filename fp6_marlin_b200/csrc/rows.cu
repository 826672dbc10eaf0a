// Row operators between the products of a decoder block: the root-mean-square norm with the residual's addition, and the
// rounding of rows to E4M3 with a scale for each 128 neighbours (with or without the norm in front).
//
//   h = x + r          in fp32; rounded once to the 16-bit type where it is stored, the norm goes on with the fp32 sum
//   y = h * rsqrt(mean(h^2) + eps) * w
//   s[g] = max(max |y| of group g, 1e-30) / 448,  q = round(y / s[g])      (NaN stays NaN in both)
//
// The reference has no counterpart; its layer lists (bench.py:53-86) name the products on either side.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>

#include "../../include/fp6m.h"
#include "host_common.h"

namespace {

using namespace fp6m;

constexpr int kGroup = 128;              // neighbours that share a scale
constexpr float kPart = 1.f / 448.f;      // of the largest magnitude: the scale.  One product, as torch on a GPU divides by a number: the same scales, bit for bit
constexpr float kSmallest = 1e-30f;

template <class T> struct Pair;
template <> struct Pair<half> {
  static __device__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<half2*>(&v)); }
  static __device__ uint32_t pack(float a, float b) { half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
};
template <> struct Pair<__nv_bfloat16> {
  static __device__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
  static __device__ uint32_t pack(float a, float b) { __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
};
template <class T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 two = Pair<T>::unpack(w[i]);
    f[2 * i] = two.x;
    f[2 * i + 1] = two.y;
  }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Pair<T>::pack(f[0], f[1]), Pair<T>::pack(f[2], f[3]), Pair<T>::pack(f[4], f[5]), Pair<T>::pack(f[6], f[7]));
}
// the larger of two, NaN if one is
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// The sum over the CTA, in one order.
__device__ __forceinline__ float sum_of_block(float sum, float* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return sum;
  if (lane == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = lane < warps ? part[lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// (N - 1 and not N + 127: rows may be as long as an int can say)
__device__ __forceinline__ int groups_of(int N) { return (N - 1) / kGroup + 1; }

// x / d, rounded once, from a reciprocal that is rounded once: the product's remainder is exact in a fused multiply-add, and what it adds makes up for the
// reciprocal's error (P. Markstein, IBM Journal of Research and Development 34, 1990).  Two values at a time: three instructions, and one reciprocal for all
// of a divisor's.  Against a multiplication by the reciprocal, which is off where a quotient lies between two E4M3 values, calls of 16384 x 8192 with the norm /
// 4099 x 11008 without take 1 / 2 % longer, with divisions 17 / 37 %.
struct Divisor {
  unsigned long long d, inverse;         // twice the same
  __device__ __forceinline__ explicit Divisor(float by) {
    d = two_of(isinf(by) ? -0.f : -by);  // (finite values by infinity are 0)
    inverse = two_of(__frcp_rn(by));
  }
  static __device__ __forceinline__ unsigned long long pack(float a, float b) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
  }
  static __device__ __forceinline__ unsigned long long two_of(float a) { return pack(a, a); }
  __device__ __forceinline__ float2 divide(float a, float b) const {
    const unsigned long long x = pack(a, b);
    unsigned long long q, rest;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(x), "l"(inverse));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(rest) : "l"(q), "l"(d), "l"(x));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q) : "l"(rest), "l"(inverse), "l"(q));
    float2 out;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(out.x), "=f"(out.y) : "l"(q));
    return out;
  }
};

struct RowParams {
  const void *x, *weight, *residual;
  void *residual_out, *y;
  float* scales;
  int M, N;
  float eps;
};

// Stores vector v of a row: in 16 bits, or in E4M3 with the scale of the 128 values that sixteen neighbouring lanes hold.  All lanes of a warp call it.
template <class T, bool kFp8>
__device__ __forceinline__ void finish_vector(const RowParams& p, size_t row, int v, int vecs, int groups, const float (&f)[8]) {
  if (kFp8) {
    float top = kSmallest;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(f[i]));
#pragma unroll
    for (int o = 8; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (v < vecs) {
      const float scale = top * kPart;
      const Divisor by(scale);
      uint2 q;
      auto two = [&](int i) { return (uint32_t)__nv_cvt_float2_to_fp8x2(by.divide(f[i], f[i + 1]), __NV_SATFINITE, __NV_E4M3); };
      q.x = two(0) | two(2) << 16;
      q.y = two(4) | two(6) << 16;
      static_cast<uint2*>(p.y)[row * vecs + v] = q;
      if (v % 16 == 0) p.scales[row * groups + v / 16] = scale;
    }
  } else if (v < vecs) {
    static_cast<uint4*>(p.y)[row * vecs + v] = pack8<T>(f);
  }
}

// One CTA a row; a thread holds kVecs groups of eight neighbouring values of it (a vector), blockDim.x vectors apart.  Every value is read once: what the
// second half of the work needs stays in registers, and the weights are on their way while the squares are summed.  Sixteen lanes hold the
// 128 values that share a scale.  Bound by memory: 16384 x 8192 with residual, fp16 to E4M3, takes 145 us in replays of a graph,
// 6.5 TB/s, which is what a plain copy reaches here, and 162 us, 5.8 TB/s, in public calls one behind the other (rows read twice, from L2 the second time: 190 us in a
// graph).  4099 x 11008 without the norm, fp16 to E4M3: 27.8 us, 4.9 TB/s, in calls; its 4099 rows of eleven warps leave a last round of CTAs a
// quarter full.  Where rows are few, what counts is latency (1 x 4096: 1.6 us in a graph, 3.0 in calls): more threads with a vector each (launch_kind).
template <class T, bool kNorm, bool kFp8, int kVecs>
__global__ void __launch_bounds__(kVecs == 4 ? 512 : 1024) rows_kernel(const RowParams p) {
  __shared__ float part[32];
  const size_t row = blockIdx.x;
  const int vecs = p.N / 8, groups = groups_of(p.N);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint4* x = static_cast<const uint4*>(p.x) + row * vecs;
  uint4 in[kVecs], add[kVecs], weight[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < vecs) in[i] = x[v];
  }
  const bool residual = kNorm && p.residual;
  if (residual) {
    const uint4* r = static_cast<const uint4*>(p.residual) + row * vecs;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < vecs) add[i] = r[v];
    }
  }
  if (kNorm) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < vecs) weight[i] = static_cast<const uint4*>(p.weight)[v];
    }
  }
  float f[kVecs][8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[i][e] = 0.f;
    if (v < vecs) {
      unpack8<T>(in[i], f[i]);
      if (residual) {
        float more[8];
        unpack8<T>(add[i], more);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] += more[e];
        static_cast<uint4*>(p.residual_out)[row * vecs + v] = pack8<T>(f[i]);
      }
    }
    if (kNorm) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += f[i][e] * f[i][e];
    }
  }
  float factor = 1.f;
  if (kNorm) factor = rsqrtf(sum_of_block(sum, part) / p.N + p.eps);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (kNorm && v < vecs) {
      float w[8];
      unpack8<T>(weight[i], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * factor * w[e];
    }
    finish_vector<T, kFp8>(p, row, v, vecs, groups, f[i]);
  }
}

// Rows of any length: every pass reads the row again (from L2, mostly).
template <class T, bool kNorm, bool kFp8>
__global__ void __launch_bounds__(1024) long_rows_kernel(const RowParams p) {
  __shared__ float part[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const size_t row = blockIdx.x;
  const int vecs = p.N / 8, groups = groups_of(p.N);
  const uint4* x = static_cast<const uint4*>(p.x) + row * vecs;
  const uint4* r = p.residual ? static_cast<const uint4*>(p.residual) + row * vecs : nullptr;
  auto load = [&](int v, float (&f)[8]) {
    unpack8<T>(x[v], f);
    if (kNorm && r) {
      float add[8];
      unpack8<T>(r[v], add);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] += add[i];
    }
  };
  float factor = 1.f;
  if (kNorm) {
    float sum = 0.f;
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
      float f[8];
      load(v, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += f[i] * f[i];
    }
    factor = rsqrtf(sum_of_block(sum, part) / p.N + p.eps);
  }
  for (int v0 = 0; v0 < vecs; v0 += blockDim.x) {
    const int v = v0 + threadIdx.x;
    float f[8] = {};
    if (v < vecs) {
      load(v, f);
      if (kNorm) {
        if (p.residual_out) static_cast<uint4*>(p.residual_out)[row * vecs + v] = pack8<T>(f);
        float w[8];
        unpack8<T>(static_cast<const uint4*>(p.weight)[v], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = f[i] * factor * w[i];
      }
    }
    finish_vector<T, kFp8>(p, row, v, vecs, groups, f);
  }
}

template <class T, bool kNorm, bool kFp8>
cudaError_t launch_kind(const RowParams& p, cudaStream_t stream) {
  const int vecs = p.N / 8;
  // Few rows (a multiprocessor gets one or two): as many threads as there are vectors, up to 1024.  Many: four vectors a thread, so that more rows are in flight
  // (16384 x 8192, norm, residual and E4M3, in a graph: 144 us; two vectors a thread 163).
  const int kind = p.M > 512 && vecs >= 128 ? 4 : vecs <= 1024 ? 1 : 2;
  const int threads = ((vecs + kind - 1) / kind + 31) / 32 * 32;
  if (vecs > 2048) return launch_overlapped(long_rows_kernel<T, kNorm, kFp8>, dim3(p.M), dim3(1024), 0, stream, p);
  return launch_overlapped(kind == 1 ? rows_kernel<T, kNorm, kFp8, 1> : kind == 2 ? rows_kernel<T, kNorm, kFp8, 2> : rows_kernel<T, kNorm, kFp8, 4>, dim3(p.M), dim3(threads), 0,
                           stream, p);
}
template <class T>
cudaError_t launch_rows(const RowParams& p, bool norm, cudaStream_t stream) {
  return !norm ? launch_kind<T, false, true>(p, stream) : p.scales ? launch_kind<T, true, true>(p, stream) : launch_kind<T, true, false>(p, stream);
}

int rows_impl(const RowParams& p, bool norm, int type, int dev, void* stream, const char* what) {
  if (p.M < 0 || p.N < 0 || p.N % 8 || (type != FP6M_TYPE_F16 && type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (p.M == 0 || p.N == 0) return FP6M_OK;
  if (!p.x || !p.y || (norm && !p.weight) || (p.residual != nullptr) != (p.residual_out != nullptr)) return FP6M_ERR_BAD_ARG;
  if (!aligned16(p.x) || !aligned16(p.weight) || !aligned16(p.residual) || !aligned16(p.residual_out) || !aligned16(p.y) ||
      (reinterpret_cast<uintptr_t>(p.scales) & 3))
    return FP6M_ERR_BAD_ARG;
  DeviceGuard guard(dev);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = type == FP6M_TYPE_F16 ? launch_rows<half>(p, norm, st) : launch_rows<__nv_bfloat16>(p, norm, st);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, what);
}

}  // namespace

extern "C" {

int fp6m_rms_norm(const void* x, const void* weight, const void* residual, void* residual_out, void* y, void* scales, int M, int N, float eps, int type,
                  int dev, void* stream) {
  RowParams p = {x, weight, residual, residual_out, y, static_cast<float*>(scales), M, N, eps};
  return rows_impl(p, true, type, dev, stream, "rms_norm launch");
}

int fp6m_quantize_fp8(const void* x, void* q, void* scales, int M, int N, int type, int dev, void* stream) {
  if (M > 0 && N > 0 && !scales) return FP6M_ERR_BAD_ARG;
  RowParams p = {x, nullptr, nullptr, nullptr, q, static_cast<float*>(scales), M, N, 0.f};
  return rows_impl(p, false, type, dev, stream, "quantize_fp8 launch");
}

}  // extern "C"
