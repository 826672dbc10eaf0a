// Shared by the kernels of the product of E4M3 matrices with scales for blocks of 128 (mul_fp8.cu, mul_fp8_rows.cu).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "device_utils.cuh"
#include "gemm_params.h"
#include "tc5_common.cuh"

namespace fp6m {

constexpr int kBlock = 128;              // values of K, and columns of C, that share a scale
constexpr int kStripBytes = kBlock * kBlock;

constexpr int kMaxFp8Ctas = 192;         // one CTA per multiprocessor
// The scratch: launch epoch and counters, then the tagged words of the kernel for few rows, then the sums of the other.  Each keeps to
// its own part: sums must not be taken for tags.
// Most rows of A of the kernel for few rows.  us, few / many (rows x K x columns): 33 x 4096 x 4096 12.1 / 11.7, 64 x 4096 x 4096 13.0 / 11.9, 48 x 11008 x 4096
// 17.5 / 20.6, 64 x 8192 x 57344 87 / 97.
constexpr int kMostColumnsRows = 64;
constexpr size_t kFp8Header = (kEpochWords + kMaxFp8Ctas) * sizeof(unsigned int);
constexpr size_t kRowsScratch = kFp8Header + (size_t)kMaxFp8Ctas * kMostColumnsRows * kBlock * sizeof(unsigned long long);

struct Fp8Args {
  const void *A, *B;
  void* C;
  const float *sa, *sb;
  int M, N, K, kb;                       // kb: blocks of K
  bool bf16;
  void* scratch;
  int* status;
};
// mul_fp8_rows.cu
size_t fp8_rows_scratch_bytes(int M, int N, int K, int sms);
cudaError_t launch_fp8_rows(const Fp8Args& a, int sms, cudaStream_t stream);

#ifdef __CUDACC__
// x (bytes of K) is a multiple of 128: the copy starts on a 16-byte boundary
__device__ __forceinline__ void tma_load_bytes(uint32_t dst, const CUtensorMap* map, int x, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_prefetch_bytes(const CUtensorMap* map, int x, int row) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(row) : "memory");
}
__device__ __forceinline__ float4 lds_float4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// Words of a partial at constant distances: their places are constants in the instructions, not registers (with an address register
// for each of 64 values the sums were spilled).
template <int kOffset>
__device__ __forceinline__ unsigned long long ld_partial(const unsigned long long* slot) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1 + %2];" : "=l"(v) : "l"(slot), "n"(kOffset * 8) : "memory");
  return v;
}
template <int kOffset>
__device__ __forceinline__ void st_partial(unsigned long long* slot, unsigned long long v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0 + %1], %2;" ::"l"(slot), "n"(kOffset * 8), "l"(v) : "memory");
}
template <int kFirst, class F, int... kI>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, kI...>) { (f(std::integral_constant<int, kFirst + kI>()), ...); }
// f(kFirst) ... f(kFirst + kCount - 1), the argument a constant
template <int kFirst, int kCount, class F>
__device__ __forceinline__ void each(F&& f) { each_of<kFirst>(f, std::make_integer_sequence<int, kCount>()); }
__device__ __forceinline__ void store_value(half* c, float v) { *c = __float2half_rn(v); }
__device__ __forceinline__ void store_value(__nv_bfloat16* c, float v) { *c = __float2bfloat16_rn(v); }
#endif  // __CUDACC__

}  // namespace fp6m
