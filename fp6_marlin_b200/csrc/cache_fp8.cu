// Tokens into and out of a paged cache in 8 bits: E4M3 values with a power of two for each token and head.
//
//   e = the least integer in lowest .. highest with max |x| <= 448 * 2^e      over the finite values of a head
//   q = round(x * 2^-e) to E4M3;  q * 2^e stands for x
//
// A power of two, and not the quotient of the largest magnitude by 448, because E4M3 is a floating-point format: where its range starts changes nothing
// for values that stay within it, so a scale between two powers gains nothing but the values that are up to a factor of two smaller than its least;
// in return q * 2^e is exact in fp16 and bf16, takes a byte, and attention needs no multiplication by it (tree_attention_fp8.cu).
// The exponents end where the 16-bit type has no finer values (fp16: 2^-15 times E4M3's least is fp16's), or nothing that a model's keys and values hold (bf16: 2^-40),
// and above, where 240 * 2^e is still finite in that type and 256 * 2^e is not: there values end at 240.
//
// The reference has no counterpart; its layer lists (bench.py:53-86) name the products on either side.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>

#include "../../include/fp6m.h"
#include "host_common.h"
#include "tree_attention.cuh"

namespace {

using namespace fp6m;

constexpr int kThreads = 256;

template <class T> struct Exponents;
template <> struct Exponents<half> { static constexpr int kLowest = -15, kHighest = 8; };
template <> struct Exponents<__nv_bfloat16> { static constexpr int kLowest = -40, kHighest = 120; };
constexpr float kMost = 448.f, kMostAtHighest = 240.f;

struct CacheParams {
  fp6m_cache_fp8_args a;
  fp6m_cache_scales s;
  unsigned long long page_magic;         // division by the page size, see tree_attention.cuh
  int page_shift;
  int at_once;                           // entries of a CTA
  int* status;
};

// Where token j of a page table's row lies: page and slot, or false.
__device__ __forceinline__ bool find(const CacheParams& p, int b, int j, int* page, int* slot) {
  const int place = (int)((unsigned long long)j * p.page_magic >> p.page_shift);
  *page = p.a.page_table[b * p.a.page_table_stride + place];
  *slot = j - place * p.a.page_size;
  return (unsigned)*page < (unsigned)p.a.pages;
}
__device__ __forceinline__ void unpack16(const uint4& lo, const uint4& hi, uint32_t (&w)[8]) {
  w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w;
  w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
}

// A thread has sixteen neighbouring values of a head: 32 bytes on one side, 16 on the other; four or eight threads a head, the heads of a token's keys, then those of its
// values, side by side.  Bound by memory where tokens are many, by four look-ups one after the other (length, list, page table, values) where they are few.
template <class T, int D, bool kWrite>
__global__ void __launch_bounds__(kThreads) cache_fp8_kernel(const __grid_constant__ CacheParams p) {
  constexpr int kPart = D / 16;
  const fp6m_cache_fp8_args& a = p.a;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int heads = 2 * a.kv_heads, per_entry = heads * kPart;
  const long long entries = (long long)a.batch * a.entries, first = (long long)blockIdx.x * p.at_once;
  const int here = (int)min((long long)p.at_once, entries - first), work = here * per_entry;
  const long long most = (long long)a.max_pages * a.page_size;
  bool bad = false;
  for (int i0 = 0; i0 < work; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    bool lives = i < work;
    const int entry_here = lives ? i / per_entry : 0, in_entry = i - entry_here * per_entry;
    const int part = i % kPart, head = in_entry / kPart % a.kv_heads;
    const bool values = in_entry / kPart >= a.kv_heads;
    const int b = (int)((first + entry_here) / a.entries), entry = (int)((first + entry_here) - (long long)b * a.entries);
    long long at = 0;
    int token = entry;
    if (lives) {
      const int length = (int)min((long long)max(a.lengths[b], 0), most);
      if (kWrite) {
        if (a.counts && entry >= a.counts[b]) lives = false;
        if (lives && a.list) token = a.list[b * a.list_stride + entry];
        lives = lives && token >= 0;
        at = (long long)length + entry;
        if (lives && (at >= most || token >= a.tokens)) {
          bad = true;
          lives = false;
        }
      } else {
        at = (long long)(a.starts ? a.starts[b] : 0) + entry;
        lives = at >= 0 && at < length;
      }
    }
    int page = 0, slot = 0;
    if (lives && !find(p, b, (int)at, &page, &slot)) {
      bad = true;
      lives = false;
    }
    const long long* wide_stride = values ? a.v_stride : a.k_stride;
    const long long* narrow_stride = values ? a.v_cache_stride : a.k_cache_stride;
    const long long* byte_stride = values ? p.s.v_scales_stride : p.s.k_scales_stride;
    T* wide = static_cast<T*>(values ? a.v : a.k) + b * wide_stride[0] + token * wide_stride[1] + head * wide_stride[2] + part * 16;
    uint8_t* narrow = static_cast<uint8_t*>(values ? a.v_cache : a.k_cache) + page * narrow_stride[0] + slot * narrow_stride[1] + head * narrow_stride[2] + part * 16;
    uint8_t* byte = static_cast<uint8_t*>(values ? p.s.v_scales : p.s.k_scales) + page * byte_stride[0] + slot * byte_stride[1] + head * byte_stride[2];
    if constexpr (kWrite) {
      uint32_t w[8] = {};
      if (lives) unpack16(reinterpret_cast<const uint4*>(wide)[0], reinterpret_cast<const uint4*>(wide)[1], w);
      float x[16], top = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[e] = Half16<T>::value((uint16_t)(w[e / 2] >> 16 * (e & 1)));
        top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
      }
#pragma unroll
      for (int o = 1; o < kPart; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // top = 1.m * 2^n; 448 = 1.75 * 2^8
      const uint32_t bits = __float_as_uint(top);
      const int least = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
      const int power = min(max(least, Exponents<T>::kLowest), Exponents<T>::kHighest);
      const float down = __uint_as_float((uint32_t)(127 - power) << 23), limit = power == Exponents<T>::kHighest ? kMostAtHighest : kMost;
      uint32_t q[4];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float two[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) two[f] = fabsf(x[e + f]) < INFINITY ? fminf(fmaxf(x[e + f] * down, -limit), limit) : __uint_as_float(0x7fc00000u);
        const uint32_t pair = __nv_cvt_float2_to_fp8x2(make_float2(two[0], two[1]), __NV_SATFINITE, __NV_E4M3);
        q[e / 4] = e & 2 ? q[e / 4] | pair << 16 : pair;
      }
      if (lives) {
        *reinterpret_cast<uint4*>(narrow) = make_uint4(q[0], q[1], q[2], q[3]);
        if (part == 0) *byte = (uint8_t)(power + 127);
      }
    } else if (lives) {
      const uint4 q = *reinterpret_cast<const uint4*>(narrow);
      const uint32_t by_bits = *byte;
      const float by = __uint_as_float(by_bits ? by_bits << 23 : 0x00400000u);
      const uint32_t in[4] = {q.x, q.y, q.z, q.w};
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(in[e / 2] >> 16 * (e & 1)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const half2*>(&two));
        w[e] = Half16<T>::pack(f.x * by, f.y * by);
      }
      reinterpret_cast<uint4*>(wide)[0] = make_uint4(w[0], w[1], w[2], w[3]);
      reinterpret_cast<uint4*>(wide)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  if (bad && p.status) atomicExch(p.status, FP6M_ERR_BAD_ARG);
}

template <class T, int D>
cudaError_t launch(const CacheParams& p, bool write, unsigned ctas, cudaStream_t stream) {
  return write ? launch_overlapped(cache_fp8_kernel<T, D, true>, dim3(ctas), dim3(kThreads), 0, stream, p)
               : launch_overlapped(cache_fp8_kernel<T, D, false>, dim3(ctas), dim3(kThreads), 0, stream, p);
}

int run(const fp6m_cache_fp8_args* args, const fp6m_cache_scales* scales, bool write, int dev, void* stream, int* status_dev) {
  if (!args || !scales) return FP6M_ERR_BAD_ARG;
  const fp6m_cache_fp8_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.entries < 0 || (a.type != FP6M_TYPE_F16 && a.type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (a.head_dim != 64 && a.head_dim != 128) return FP6M_ERR_PROB_SHAPE;
  if (a.batch == 0 || a.entries == 0 || a.kv_heads == 0) return FP6M_OK;
  if (a.kv_heads < 0 || a.kv_heads > 1 << 24 || a.max_pages < 0 || a.pages < 0 || a.page_size <= 0 || (long long)a.max_pages * a.page_size > 0x7fff0000ll) return FP6M_ERR_PROB_SHAPE;
  if (!a.lengths || a.list_stride < 0 || !rows_aligned(a.k, a.k_stride, 8) || !rows_aligned(a.v, a.v_stride, 8)) return FP6M_ERR_BAD_ARG;
  if (a.max_pages > 0) {
    if (!rows_aligned(a.k_cache, a.k_cache_stride, 16) || !rows_aligned(a.v_cache, a.v_cache_stride, 16) || !a.page_table || a.page_table_stride < 0) return FP6M_ERR_BAD_ARG;
    if (!scales->k_scales || !scales->v_scales) return FP6M_ERR_BAD_ARG;
    for (int i = 0; i < 3; ++i)
      if (scales->k_scales_stride[i] < 0 || scales->v_scales_stride[i] < 0) return FP6M_ERR_BAD_ARG;
  }
  DeviceGuard guard(dev);
  CacheParams p;
  p.a = a;
  p.s = *scales;
  p.status = status_dev;
  division_by(a.page_size, &p.page_magic, &p.page_shift);
  const int per_entry = 2 * a.kv_heads * (a.head_dim / 16);
  p.at_once = per_entry >= kThreads ? 1 : kThreads / per_entry;
  const long long ctas = ((long long)a.batch * a.entries + p.at_once - 1) / p.at_once;
  if (ctas > INT_MAX) return FP6M_ERR_PROB_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool is_half = a.type == FP6M_TYPE_F16;
  const cudaError_t e = a.head_dim == 64 ? (is_half ? launch<half, 64>(p, write, (unsigned)ctas, st) : launch<__nv_bfloat16, 64>(p, write, (unsigned)ctas, st))
                                         : (is_half ? launch<half, 128>(p, write, (unsigned)ctas, st) : launch<__nv_bfloat16, 128>(p, write, (unsigned)ctas, st));
  return e == cudaSuccess ? FP6M_OK : cuda_fail(e, "cache_fp8 launch");
}

}  // namespace

extern "C" {

int fp6m_write_cache_fp8(const fp6m_cache_fp8_args* args, const fp6m_cache_scales* scales, int dev, void* stream, int* status_dev) {
  return run(args, scales, true, dev, stream, status_dev);
}
int fp6m_read_cache_fp8(const fp6m_cache_fp8_args* args, const fp6m_cache_scales* scales, int dev, void* stream, int* status_dev) {
  return run(args, scales, false, dev, stream, status_dev);
}

}  // extern "C"
