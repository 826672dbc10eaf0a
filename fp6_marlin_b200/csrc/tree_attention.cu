// Attention of T drafted tokens of each of B sequences over a paged cache of committed tokens and the drafted tokens themselves.
//
//   o_i = sum_j p_ij v_j,   p_i = softmax_j(scale * q_i . k_j)
//
// over the lengths[b] cached tokens and the drafted tokens j whose bit is set in the mask of i.  A mask of zero marks padding:
// it sees nothing and gives zeros.  The reference has no counterpart; its layer lists (bench.py:53-86) name the products on either side.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/fp6m.h"
#include "host_common.h"

namespace {

using namespace fp6m;

__device__ __forceinline__ float to_float(half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store(half* c, float v) { *c = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* c, float v) { *c = __float2bfloat16_rn(v); }

// One warp a query, a key at a time.
template <class T, int D>
__global__ void __launch_bounds__(128) tree_attention_plain_kernel(const fp6m_tree_attention_args a, int* status) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long query = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (query >= (long long)a.batch * a.tokens * a.heads) return;
  const int h = (int)(query % a.heads), t = (int)(query / a.heads % a.tokens), b = (int)(query / a.heads / a.tokens);
  const int g = h / (a.heads / a.kv_heads);
  constexpr int E = D / 32;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + h * a.q_stride[2];
  float qf[E], o[E] = {}, top = -INFINITY, total = 0.f;
  for (int i = 0; i < E; ++i) qf[i] = to_float(q[lane + 32 * i]) * a.scale;
  const unsigned long long mask = static_cast<const unsigned long long*>(a.tree)[b * a.tree_stride + t];
  const int capacity = a.max_pages * a.page_size;
  int length = static_cast<const int*>(a.lengths)[b];
  length = length < 0 ? 0 : length > capacity ? capacity : length;
  auto visit = [&](const T* k, const T* v) {
    float s = 0.f;
    for (int i = 0; i < E; ++i) s += qf[i] * to_float(k[lane + 32 * i]);
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float now = fmaxf(top, s);
    if (now == -INFINITY) return;
    const float keep = __expf(top - now), p = __expf(s - now);
    total = total * keep + p;
    for (int i = 0; i < E; ++i) o[i] = o[i] * keep + p * to_float(v[lane + 32 * i]);
    top = now;
  };
  if (mask) {
    for (int j = 0; j < length; ++j) {
      const int page = static_cast<const int*>(a.page_table)[b * a.page_table_stride + j / a.page_size];
      if (page < 0 || page >= a.pages) {
        if (lane == 0 && status) atomicExch(status, FP6M_ERR_BAD_ARG);
        continue;
      }
      const long long slot = j % a.page_size;
      visit(static_cast<const T*>(a.k_cache) + page * a.k_cache_stride[0] + slot * a.k_cache_stride[1] + g * a.k_cache_stride[2],
            static_cast<const T*>(a.v_cache) + page * a.v_cache_stride[0] + slot * a.v_cache_stride[1] + g * a.v_cache_stride[2]);
    }
    for (int j = 0; j < a.tokens; ++j)
      if (mask >> j & 1)
        visit(static_cast<const T*>(a.k) + b * a.k_stride[0] + j * a.k_stride[1] + g * a.k_stride[2],
              static_cast<const T*>(a.v) + b * a.v_stride[0] + j * a.v_stride[1] + g * a.v_stride[2]);
  }
  T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + t * a.out_stride[1] + h * a.out_stride[2];
  for (int i = 0; i < E; ++i) store(out + lane + 32 * i, total > 0.f ? o[i] / total : total == total ? 0.f : total);
}

template <class T>
cudaError_t launch_tree(const fp6m_tree_attention_args& a, cudaStream_t stream, int* status) {
  const long long warps = (long long)a.batch * a.tokens * a.heads;
  return launch_overlapped(a.head_dim == 64 ? tree_attention_plain_kernel<T, 64> : tree_attention_plain_kernel<T, 128>, dim3((unsigned)((warps + 3) / 4)), dim3(128),
                           0, stream, a, status);
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

size_t fp6m_tree_attention_scratch_bytes(int sms) { return 256; }

int fp6m_tree_attention(const fp6m_tree_attention_args* args, void* scratch, size_t scratch_bytes, int dev, void* stream, int* status_dev) {
  if (!args) return FP6M_ERR_BAD_ARG;
  const fp6m_tree_attention_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.heads < 0 || (a.type != FP6M_TYPE_F16 && a.type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (a.tokens > 64 || (a.head_dim != 64 && a.head_dim != 128)) return FP6M_ERR_PROB_SHAPE;
  if (a.batch == 0 || a.tokens == 0 || a.heads == 0) return FP6M_OK;
  if (a.kv_heads <= 0 || a.heads % a.kv_heads) return FP6M_ERR_PROB_SHAPE;
  if (a.max_pages < 0 || a.pages < 0 || a.page_size <= 0 || (long long)a.max_pages * a.page_size > 0x7fffff00ll) return FP6M_ERR_PROB_SHAPE;
  if ((long long)a.batch * a.tokens * a.heads > 0x7fffffffll) return FP6M_ERR_PROB_SHAPE;
  if (!rows_aligned(a.q, a.q_stride) || !rows_aligned(a.k, a.k_stride) || !rows_aligned(a.v, a.v_stride) || !rows_aligned(a.out, a.out_stride)) return FP6M_ERR_BAD_ARG;
  if (!a.lengths || !a.tree || a.tree_stride < 0) return FP6M_ERR_BAD_ARG;
  if (a.max_pages > 0 && (!rows_aligned(a.k_cache, a.k_cache_stride) || !rows_aligned(a.v_cache, a.v_cache_stride) || !a.page_table || a.page_table_stride < 0)) return FP6M_ERR_BAD_ARG;
  DeviceGuard guard(dev);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.type == FP6M_TYPE_F16 ? launch_tree<half>(a, st, status_dev) : launch_tree<__nv_bfloat16>(a, st, status_dev);
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "tree_attention launch");
}

}  // extern "C"
