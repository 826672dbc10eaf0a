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

#include <algorithm>

#include "../../include/fp6m.h"
#include "host_common.h"
#include "tree_attention.cuh"

namespace {

using namespace fp6m;

constexpr int kThreads = 256;

constexpr float kMostAtHighest = 240.f;

// What depends on the type: the exponents, and sixteen values at a time to and from E4M3.
template <class T> struct Values;
template <> struct Values<half> {
  using Two = half2;
  static constexpr int kLowest = -15, kHighest = 8;
  // The products are exact, or so small that they become E4M3's zero.
  static __device__ __forceinline__ void narrow(const uint32_t (&w)[8], int exponent, uint32_t (&q)[4]) {
    const half2 by = __half2half2(__ushort_as_half((uint16_t)((15 - exponent) << 10)));
    uint32_t pair[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      half2 x = __hmul2(*reinterpret_cast<const half2*>(&w[e]), by);
      if (exponent == kHighest) x = __hmax2(__hmin2(x, __half2half2(__float2half_rn(kMostAtHighest))), __half2half2(__float2half_rn(-kMostAtHighest)));
      pair[e] = __nv_cvt_halfraw2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = pair[2 * e] | pair[2 * e + 1] << 16;
  }
};
template <> struct Values<__nv_bfloat16> {
  using Two = __nv_bfloat162;
  static constexpr int kLowest = -40, kHighest = 120;
  static __device__ __forceinline__ void narrow(const uint32_t (&w)[8], int exponent, uint32_t (&q)[4]) {
    const uint32_t one = (uint32_t)(127 - exponent) << 7, both = one | one << 16;
    uint32_t pair[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const __nv_bfloat162 scaled = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]), *reinterpret_cast<const __nv_bfloat162*>(&both));      // (exact)
      const uint32_t v = *reinterpret_cast<const uint32_t*>(&scaled);
      float x = __uint_as_float(v << 16), y = __uint_as_float(v & 0xffff0000u);
      if (exponent == kHighest) x = fminf(fmaxf(x, -kMostAtHighest), kMostAtHighest), y = fminf(fmaxf(y, -kMostAtHighest), kMostAtHighest);
      pair[e] = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = pair[2 * e] | pair[2 * e + 1] << 16;
  }
};
// The larger magnitudes of two pairs, NaN where there is one.
__device__ __forceinline__ half2 larger(half2 a, half2 b) { return __hmax2_nan(a, __habs2(b)); }
__device__ __forceinline__ __nv_bfloat162 larger(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, __habs2(b)); }

struct CacheParams {
  fp6m_cache_fp8_args a;
  fp6m_cache_scales s;
  unsigned long long page_magic;         // division by the page size, see tree_attention.cuh
  int page_shift;
  int at_once;                           // entries of a CTA
  unsigned int entry_magic;              // division by an entry's units: n * magic >> 32, exact for n * units < 2^32
  int* status;
};

// A CTA has some entries of a sequence, their keys or their values.  A unit is sixteen neighbouring values of a head: 32 bytes on one side, 16 on the other; four or eight units a
// head, the heads of a token side by side.  A thread has a unit a round; where the next one lies is looked up while this one's values are on their way.
// Writing 4 x 4096 tokens of 8 heads of 128 from bf16: 22.1 us, 4.6 TB/s; reading 16 times up to 6144 of them: 54.0 us, 5.6 TB/s: of what a copy reaches 0.70 and 0.86, the rest is the start of a
// CTA (its length, then its page, then its values), for short calls all there is: 16 x 7 tokens of 32 heads 2.4 us.  Not kept: 2, 3 and 4 units of a thread in flight together (23.3, 25.2, 27.3 and 60.8, 59.6,
// 64.4 us: registers that warps lack); accesses of 32 bytes (23.2, 62.1 of 23.3, 60.8); units of eight values (45 and 107: a head's address and power twice as often).
struct Place {
  bool lives;
  int token, page, slot, head;
};
template <class T, int D, bool kWrite>
__global__ void __launch_bounds__(kThreads) cache_fp8_kernel(const __grid_constant__ CacheParams p) {
  constexpr int kPart = D / 16;
  const fp6m_cache_fp8_args& a = p.a;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y + (blockIdx.z >> 1) * gridDim.y;
  if (b >= a.batch) return;
  const bool values = blockIdx.z & 1;
  const long long* wide_stride = values ? a.v_stride : a.k_stride;
  const long long* narrow_stride = values ? a.v_cache_stride : a.k_cache_stride;
  const long long* power_stride = values ? p.s.v_scales_stride : p.s.k_scales_stride;
  T* const wide_rows = static_cast<T*>(values ? a.v : a.k) + b * wide_stride[0];
  uint8_t* const narrow_rows = static_cast<uint8_t*>(values ? a.v_cache : a.k_cache);
  uint8_t* const powers = static_cast<uint8_t*>(values ? p.s.v_scales : p.s.k_scales);
  // (strides of tokens, pages and slots fit 32 bits)
  const unsigned wide_step = (unsigned)wide_stride[1], page_step = (unsigned)narrow_stride[0], slot_step = (unsigned)narrow_stride[1], power_page = (unsigned)power_stride[0], power_slot = (unsigned)power_stride[1];
  const long long wide_head = wide_stride[2], narrow_head = narrow_stride[2], power_head = power_stride[2];
  const int per_entry = a.kv_heads * kPart, first = blockIdx.x * p.at_once, work = min(p.at_once, a.entries - first) * per_entry;
  const int most = a.max_pages * a.page_size, length = min(max(a.lengths[b], 0), most), count = kWrite && a.counts ? a.counts[b] : a.entries;
  const unsigned start = kWrite ? length : a.starts ? a.starts[b] : 0;      // (modulo 2^32: tokens before the first come behind all)
  const int* table = a.page_table + b * a.page_table_stride;
  const int part = threadIdx.x % kPart;
  bool bad = false;
  // where unit i of this CTA comes from or goes to
  auto look_up = [&](int i) {
    Place at;
    const int in_cta = p.at_once == 1 ? 0 : (int)__umulhi((unsigned)i, p.entry_magic), entry = first + in_cta;
    at.head = (i - in_cta * per_entry) / kPart;
    at.lives = i < work;
    at.token = entry;
    const unsigned j = start + entry;
    if (kWrite) {
      at.lives = at.lives && entry < count;
      if (at.lives && a.list) at.token = a.list[b * a.list_stride + entry];
      at.lives = at.lives && at.token >= 0;
      if (at.lives && (j >= (unsigned)most || at.token >= a.tokens)) {
        bad = true;
        at.lives = false;
      }
    } else {
      at.lives = at.lives && j < (unsigned)length;
    }
    const int place = (int)((unsigned long long)j * (unsigned)p.page_magic >> p.page_shift);      // (the magic number is below 2^32)
    at.slot = (int)j - place * a.page_size;
    at.page = at.lives ? table[place] : 0;
    return at;
  };
  Place next = look_up(threadIdx.x);
#pragma unroll 1
  for (int i0 = 0; i0 < work; i0 += kThreads) {
    Place at = next;
    if (i0 + kThreads < work) next = look_up(i0 + kThreads + threadIdx.x);
    if (at.lives && (unsigned)at.page >= (unsigned)a.pages) {
      bad = true;
      at.lives = false;
    }
    uint4* const wide = reinterpret_cast<uint4*>(wide_rows + (unsigned long long)(unsigned)at.token * wide_step + at.head * wide_head + part * 16);
    uint4* const narrow = reinterpret_cast<uint4*>(narrow_rows + (unsigned long long)(unsigned)at.page * page_step + (unsigned long long)(unsigned)at.slot * slot_step + at.head * narrow_head + part * 16);
    uint8_t* const power = powers + (unsigned long long)(unsigned)at.page * power_page + (unsigned long long)(unsigned)at.slot * power_slot + at.head * power_head;
    if constexpr (kWrite) {
      uint4 in[2] = {};
      if (at.lives) {
        in[0] = wide[0];
        in[1] = wide[1];
      }
      constexpr uint32_t E = Half16<T>::kExponent;
      uint32_t w[8] = {in[0].x, in[0].y, in[0].z, in[0].w, in[1].x, in[1].y, in[1].z, in[1].w};
      using Two = typename Values<T>::Two;
      uint32_t two = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Two now = larger(*reinterpret_cast<const Two*>(&two), *reinterpret_cast<const Two*>(&w[e]));
        two = *reinterpret_cast<const uint32_t*>(&now);
      }
      two &= 0x7fff7fffu;
      uint32_t top = max(two & 0xffffu, two >> 16), odd = 0;         // (bits of magnitudes are ordered as they are); a bit for each value that is infinite or NaN
      if (top >= E) {
        // these become NaN, and the exponent is that of the others
        top = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t one = w[e / 2] >> 16 * (e & 1) & 0x7fffu;
          if (one >= E) odd |= 1u << e;
          else top = max(top, one);
        }
      }
#pragma unroll
      for (int o = 1; o < kPart; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      // = 1.m * 2^n; 448 = 1.75 * 2^8
      const uint32_t bits = __float_as_uint(Half16<T>::value((uint16_t)top));
      const int least = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
      const int exponent = min(max(least, Values<T>::kLowest), Values<T>::kHighest);
      uint32_t q[4];
      Values<T>::narrow(w, exponent, q);
      if (odd) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (odd >> e & 1) q[e / 4] |= 0x7fu << 8 * (e & 3);
      }
      if (at.lives) {
        *narrow = make_uint4(q[0], q[1], q[2], q[3]);
        if (part == 0) *power = (uint8_t)(exponent + 127);
      }
    } else {
      if (!at.lives) continue;
      const uint4 in = *narrow;
      const uint32_t by = *power;
      const float f = __uint_as_float(by ? by << 23 : 0x00400000u);
      const uint32_t q[4] = {in.x, in.y, in.z, in.w};
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q[e / 2] >> 16 * (e & 1)), __NV_E4M3);
        const float2 v = __half22float2(*reinterpret_cast<const half2*>(&two));
        w[e] = Half16<T>::pack(v.x * f, v.y * f);
      }
      wide[0] = make_uint4(w[0], w[1], w[2], w[3]);
      wide[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  if (bad && p.status) atomicExch(p.status, FP6M_ERR_BAD_ARG);
}

template <class T, int D>
cudaError_t launch(const CacheParams& p, bool write, dim3 ctas, cudaStream_t stream) {
  return write ? launch_overlapped(cache_fp8_kernel<T, D, true>, ctas, dim3(kThreads), 0, stream, p) : launch_overlapped(cache_fp8_kernel<T, D, false>, ctas, dim3(kThreads), 0, stream, p);
}

int run(const fp6m_cache_fp8_args* args, const fp6m_cache_scales* scales, bool write, int dev, void* stream, int* status_dev) {
  if (!args || !scales) return FP6M_ERR_BAD_ARG;
  const fp6m_cache_fp8_args& a = *args;
  if (a.batch < 0 || a.tokens < 0 || a.entries < 0 || (a.type != FP6M_TYPE_F16 && a.type != FP6M_TYPE_BF16)) return FP6M_ERR_BAD_ARG;
  if (a.head_dim != 64 && a.head_dim != 128) return FP6M_ERR_PROB_SHAPE;
  if (a.batch == 0 || a.entries == 0 || a.kv_heads == 0) return FP6M_OK;
  if (a.kv_heads < 0 || a.kv_heads > 1 << 16 || a.max_pages < 0 || a.pages < 0 || a.page_size <= 0 || (long long)a.max_pages * a.page_size > 0x7fff0000ll) return FP6M_ERR_PROB_SHAPE;
  if (!a.lengths || a.list_stride < 0) return FP6M_ERR_BAD_ARG;
  if (!(write && a.tokens == 0) && (!rows_aligned(a.k, a.k_stride, 8) || !rows_aligned(a.v, a.v_stride, 8))) return FP6M_ERR_BAD_ARG;      // (of no tokens nothing is read)
  if (a.max_pages > 0) {
    if (!rows_aligned(a.k_cache, a.k_cache_stride, 16) || !rows_aligned(a.v_cache, a.v_cache_stride, 16) || !a.page_table || a.page_table_stride < 0) return FP6M_ERR_BAD_ARG;
    if (!scales->k_scales || !scales->v_scales) return FP6M_ERR_BAD_ARG;
    for (int i = 0; i < 3; ++i)
      if (scales->k_scales_stride[i] < 0 || scales->v_scales_stride[i] < 0) return FP6M_ERR_BAD_ARG;
  }
  constexpr long long kStep = 0xffffffffll;          // of tokens, pages and slots
  if (a.k_stride[1] > kStep || a.v_stride[1] > kStep) return FP6M_ERR_PROB_SHAPE;
  for (int i = 0; i < 2; ++i)
    if (a.k_cache_stride[i] > kStep || a.v_cache_stride[i] > kStep || scales->k_scales_stride[i] > kStep || scales->v_scales_stride[i] > kStep) return FP6M_ERR_PROB_SHAPE;
  DeviceGuard guard(dev);
  CacheParams p;
  p.a = a;
  p.s = *scales;
  p.status = status_dev;
  division_by(a.page_size, &p.page_magic, &p.page_shift);
  const int sms = sm_count(dev);
  if (sms <= 0) return cuda_fail(cudaGetLastError(), "cudaDeviceGetAttribute");
  // A CTA goes round once for every two times that the multiprocessors are full of such, six times at most.  us with 1 / 2 / 4 / 6 / 8 rounds: reading 16 x 6144 tokens of 8 heads of 128 (41 times full)
  // 77.2 / 61.4 / 55.0 / 54.0 / 54.3; 4 x 4096 of 64 (3.5) 11.9 / 11.8 / 12.0 / 15.1 / 15.6; writing 4 x 4096 of 128 (6.9) 23.9 / 22.1 / 22.1 / 23.8 / 25.2; 8 x 512 (1.7) 7.3 / 7.6 / 9.2 / 10.5 / 11.5.
  const int per_entry = a.kv_heads * (a.head_dim / 16);
  const long long full = 2ll * a.batch * a.entries * per_entry / ((long long)sms * 8 * kThreads);
  p.at_once = (int)std::max(1ll, std::min(full / 2, 6ll)) * kThreads / per_entry;
  if (p.at_once < 1) p.at_once = 1;
  p.entry_magic = (unsigned int)((1ull << 32) / per_entry + 1);
  const dim3 ctas((unsigned)((a.entries + (long long)p.at_once - 1) / p.at_once), (unsigned)(a.batch < 65535 ? a.batch : 65535), (unsigned)(2 * ((a.batch + 65534ll) / 65535)));      // keys and values
  if (ctas.z > 65535) return FP6M_ERR_PROB_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool is_half = a.type == FP6M_TYPE_F16;
  const cudaError_t e = a.head_dim == 64 ? (is_half ? launch<half, 64>(p, write, ctas, st) : launch<__nv_bfloat16, 64>(p, write, ctas, st))
                                         : (is_half ? launch<half, 128>(p, write, ctas, st) : launch<__nv_bfloat16, 128>(p, write, ctas, st));
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
