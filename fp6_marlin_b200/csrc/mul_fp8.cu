// C[m, n] = sum over blocks b of 128 values of K:  sa[m, b] * sb[n / 128, b] * sum_k A[m, k] * B[n, k]
//
// A (M x K) and B (N x K) in E4M3, fp32 scales, fp32 sums, C in fp16 or bf16 with one rounding.
// The reference has no counterpart: its weights have four or six bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/fp6m.h"
#include "host_common.h"

namespace {

using namespace fp6m;

constexpr int kBlock = 128;      // values of K, and columns of B, that share a scale

struct Fp8Params {
  const uint8_t *A, *B;
  void* C;
  const float *sa, *sb;
  int M, N, K, kb;
};

__device__ __forceinline__ void store(half* c, float v) { *c = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* c, float v) { *c = __float2bfloat16_rn(v); }

// 32 x 64 results a CTA, 2 x 4 a thread, on plain fp32 arithmetic
template <class T>
__global__ void __launch_bounds__(256) mul_fp8_plain_kernel(const Fp8Params p) {
  constexpr int TM = 32, TN = 64, TK = 32;
  __shared__ float as[TK][TM + 1], bs[TK][TN + 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float sum[2][4] = {};
  for (int b = 0; b < p.kb; ++b) {
    float part[2][4] = {};
    for (int k0 = b * kBlock; k0 < p.K && k0 < (b + 1) * kBlock; k0 += TK) {
      __syncthreads();
      for (int i = threadIdx.x; i < (TM + TN) * TK; i += 256) {
        const int k = i % TK, r = i / TK;
        const bool is_a = r < TM;
        const int row = is_a ? m0 + r : n0 + r - TM;
        float v = 0.f;
        if (row < (is_a ? p.M : p.N) && k0 + k < p.K) {
          __nv_fp8_e4m3 e;
          e.__x = (is_a ? p.A : p.B)[(size_t)row * p.K + k0 + k];
          v = (float)e;
        }
        if (is_a) as[k][r] = v; else bs[k][r - TM] = v;
      }
      __syncthreads();
      for (int k = 0; k < TK; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] += as[k][ty * 2 + i] * bs[k][tx + 16 * j];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + ty * 2 + i, n = n0 + tx + 16 * j;
        if (m < p.M && n < p.N) sum[i][j] += part[i][j] * (p.sa[(size_t)m * p.kb + b] * p.sb[(size_t)(n / kBlock) * p.kb + b]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 2 + i, n = n0 + tx + 16 * j;
      if (m < p.M && n < p.N) store(static_cast<T*>(p.C) + (size_t)m * p.N + n, sum[i][j]);
    }
}

}  // namespace

extern "C" int fp6m_mul_fp8(const void* A, const void* B, void* C, const void* sa, const void* sb, int M, int N, int K, int type, void* scratch,
                            size_t scratch_bytes, int dev, void* stream, int* status_dev) {
  if (M < 0 || N < 0 || K < 0 || (type != FP6M_TYPE_F16 && type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (K % 16 || N % 8) return FP6M_ERR_PROB_SHAPE;
  if (M == 0 || N == 0) return FP6M_OK;
  if (!C || !aligned16(C)) return FP6M_ERR_BAD_ARG;
  DeviceGuard guard(dev);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) {                          // an empty sum
    const cudaError_t e = cudaMemsetAsync(C, 0, (size_t)M * N * 2, st);
    return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "mul_fp8 of no terms");
  }
  if (!A || !B || !sa || !sb || !aligned16(A) || !aligned16(B) || ((reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sb)) & 3)) return FP6M_ERR_BAD_ARG;
  const Fp8Params p = {static_cast<const uint8_t*>(A), static_cast<const uint8_t*>(B), C, static_cast<const float*>(sa), static_cast<const float*>(sb),
                       M, N, K, (K + kBlock - 1) / kBlock};
  const dim3 grid((N + 63) / 64, (M + 31) / 32);
  if (grid.y > 65535) return FP6M_ERR_PROB_SHAPE;
  const cudaError_t e = type == FP6M_TYPE_F16 ? launch_overlapped(mul_fp8_plain_kernel<half>, grid, dim3(256), 0, st, p)
                                              : launch_overlapped(mul_fp8_plain_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "mul_fp8 launch");
}

extern "C" size_t fp6m_mul_fp8_scratch_bytes(int M, int N, int K, int sms) { return 256; }
