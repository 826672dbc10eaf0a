// The Python call path of mul / mul_fused and of the operators between the products: reads the tensors' metadata, checks it and calls the C ABI (include/fp6m.h).
//
// A decode step is a chain of GEMMs of a few microseconds each, so the host time of a call counts: through Python
// attributes and ctypes a call took 11 us, of which the launch itself is about two.  This module handles the calls whose
// arguments are plain CUDA tensors that pass every check; for anything else - subclasses, wrappers of function
// transforms, wrong sizes or types - it answers "not handled" and the caller takes its general path, which raises or
// computes as before.  It holds no state but the addresses of the scratch buffers registered by the caller (one per device and
// stream); the caller never frees a registered buffer, also not one that a larger one replaces: a call may have read its
// address here and not have launched yet.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <type_traits>
#include <unordered_map>

#include "../../include/fp6m.h"

namespace {

// (the types of the C ABI's own declarations: the addresses come as numbers, see bind)
using MulFn = decltype(&fp6m_mul);
using MulFusedFn = decltype(&fp6m_mul_fused);
using ScratchFn = decltype(&fp6m_mul_scratch_bytes);

MulFn g_mul = nullptr;
MulFusedFn g_mul_fused = nullptr;
ScratchFn g_scratch_bytes = nullptr;

decltype(&fp6m_rms_norm) g_rms_norm = nullptr;
decltype(&fp6m_quantize_fp8) g_quantize_fp8 = nullptr;
decltype(&fp6m_mul_fp8) g_mul_fp8 = nullptr;
decltype(&fp6m_mul_fp8_scratch_bytes) g_mul_fp8_scratch_bytes = nullptr;
decltype(&fp6m_tree_attention) g_tree_attention = nullptr;
decltype(&fp6m_tree_attention_scratch_bytes) g_tree_attention_scratch_bytes = nullptr;
decltype(&fp6m_write_cache_fp8) g_write_cache_fp8 = nullptr;
decltype(&fp6m_read_cache_fp8) g_read_cache_fp8 = nullptr;
decltype(&fp6m_tree_attention_fp8) g_tree_attention_fp8 = nullptr;
decltype(&fp6m_tree_attention_fp8_scratch_bytes) g_tree_attention_fp8_scratch_bytes = nullptr;
decltype(&fp6m_verify_drafts) g_verify_drafts = nullptr;

constexpr long kNotHandled = -1;

// What the caller registered (all access under the interpreter lock).
struct Scratch {
  void* ptr;
  size_t bytes;
};
struct StreamKey {
  int dev;
  void* stream;
  bool operator==(const StreamKey& o) const { return dev == o.dev && stream == o.stream; }
};
struct StreamKeyHash {
  size_t operator()(const StreamKey& k) const { return std::hash<void*>()(k.stream) * 31 + (size_t)k.dev; }
};
// of the GEMMs, of mul_fp8, of tree_attention, of tree_attention_fp8
enum { kOfGemms = 0, kOfMulFp8 = 1, kOfTreeAttention = 2, kOfTreeAttentionFp8 = 3, kOwners = 4 };
std::unordered_map<StreamKey, Scratch, StreamKeyHash>& scratches(int owner = kOfGemms) {
  static auto* m = new std::unordered_map<StreamKey, Scratch, StreamKeyHash>[kOwners];
  return m[owner];
}
struct Device {
  int* status = nullptr;
  int sms = 0;
};
Device g_devices[64];

// A tensor whose memory may be handed to a kernel directly: a plain torch.Tensor / Parameter, strided and on a CUDA device, none of torch's
// wrappers.
const at::Tensor* plain_strided(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined()) return nullptr;
  // the keys every strided CUDA tensor may have; wrappers, conjugate views and the like have others
  static const c10::DispatchKeySet kPlain = c10::DispatchKeySet(c10::DispatchKey::CUDA) |
                                            c10::getAutogradRelatedKeySetFromBackend(c10::BackendComponent::CUDABit) |
                                            c10::getAutocastRelatedKeySetFromBackend(c10::BackendComponent::CUDABit);
  if ((t.key_set().raw_repr() & ~kPlain.raw_repr()) != 0 || !t.is_cuda()) return nullptr;
  return &t;
}
// ... and contiguous
const at::Tensor* plain_cuda(PyObject* o) {
  const at::Tensor* t = plain_strided(o);
  return t && t->is_contiguous() ? t : nullptr;
}

bool as_int(PyObject* o, int* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow || v < INT32_MIN || v > INT32_MAX) return false;
  *out = (int)v;
  return true;
}

// mul(A, B, C, s, workspace, quant_cols, thread_k, thread_n, sms, max_par, group_size, epilogue, residual) -> the C ABI's
// status, or -1: not handled.
PyObject* mul_impl(PyObject* const* args) {
  const at::Tensor* A = plain_cuda(args[0]);
  const at::Tensor* B = plain_cuda(args[1]);
  const at::Tensor* C = plain_cuda(args[2]);
  const at::Tensor* s = plain_cuda(args[3]);
  const at::Tensor* ws = plain_cuda(args[4]);
  int quant_cols, thread_k, thread_n, sms, max_par, group_size, epilogue;
  if (!A || !B || !C || !s || !ws || !as_int(args[5], &quant_cols) || !as_int(args[6], &thread_k) || !as_int(args[7], &thread_n) ||
      !as_int(args[8], &sms) || !as_int(args[9], &max_par) || !as_int(args[10], &group_size) || !as_int(args[11], &epilogue))
    return PyLong_FromLong(kNotHandled);
  if (A->dim() != 2 || C->dim() != 2) return PyLong_FromLong(kNotHandled);
  const int64_t M = A->size(0), K = A->size(1), N = C->size(1) * (epilogue == FP6M_EPILOGUE_SILU_MUL ? 2 : 1);
  if (M <= 0 || K <= 0 || N <= 0 || M > INT32_MAX || K > INT32_MAX || N > INT32_MAX || C->size(0) != M || max_par < 1) return PyLong_FromLong(kNotHandled);
  if (ws->numel() < N / 128 * max_par) return PyLong_FromLong(kNotHandled);
  if (A->scalar_type() != at::kHalf || C->scalar_type() != at::kHalf || s->scalar_type() != at::kHalf) return PyLong_FromLong(kNotHandled);
  const void* residual = nullptr;
  if (epilogue == FP6M_EPILOGUE_RESIDUAL) {
    const at::Tensor* r = plain_cuda(args[12]);
    if (!r || r->scalar_type() != at::kHalf || r->dim() != 2 || r->size(0) != M || r->size(1) != N) return PyLong_FromLong(kNotHandled);
    residual = r->data_ptr();
  }
  const int dev = A->device().index();
  if (dev < 0 || dev >= 64 || !g_devices[dev].status) return PyLong_FromLong(kNotHandled);
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const auto it = scratches().find({dev, stream});
  if (it == scratches().end()) return PyLong_FromLong(kNotHandled);
  if (it->second.bytes < g_scratch_bytes((int)M, (int)N, (int)K, quant_cols, g_devices[dev].sms)) return PyLong_FromLong(kNotHandled);
  const void *a = A->data_ptr(), *w = B->data_ptr(), *sc = s->data_ptr();
  void *c = C->data_ptr(), *wsp = ws->data_ptr();
  const size_t ws_bytes = (size_t)ws->numel() * ws->element_size();
  const Scratch scratch = it->second;
  int* status = g_devices[dev].status;
  int rc;
  Py_BEGIN_ALLOW_THREADS        // a launch waits while the GPU's queue is full
  if (epilogue)
    rc = g_mul_fused(a, w, c, sc, (int)M, (int)N, (int)K, wsp, ws_bytes, scratch.ptr, scratch.bytes, dev, stream, thread_k, thread_n, sms, max_par,
                     quant_cols, group_size, FP6M_LAYOUT_B200, status, epilogue, residual);
  else
    rc = g_mul(a, w, c, sc, (int)M, (int)N, (int)K, wsp, ws_bytes, scratch.ptr, scratch.bytes, dev, stream, thread_k, thread_n, sms, max_par,
               quant_cols, group_size, FP6M_LAYOUT_B200, status);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// ---- the operators between the products: the C ABI's status, or -1: not handled -----------------------------------------------

constexpr int kGroup = 128;            // neighbours that share a scale

bool type_of(const at::Tensor& t, int* type) {
  if (t.scalar_type() == at::kHalf) *type = FP6M_TYPE_F16;
  else if (t.scalar_type() == at::kBFloat16) *type = FP6M_TYPE_BF16;
  else return false;
  return true;
}
bool is_matrix(const at::Tensor* t, int64_t rows, int64_t columns, at::ScalarType type, int dev) {
  return t && t->dim() == 2 && t->size(0) == rows && t->size(1) == columns && t->scalar_type() == type && t->device().index() == dev;
}
bool as_float(PyObject* o, float* out) {
  if (!PyFloat_CheckExact(o)) return false;
  *out = (float)PyFloat_AS_DOUBLE(o);
  return true;
}

// rms_norm(x, weight, y, eps, scales, residual, residual_out); quantize_fp8(x, q, scales) is the same without weight
PyObject* rows_impl(PyObject* x_arg, PyObject* weight_arg, PyObject* y_arg, PyObject* eps_arg, PyObject* scales_arg, PyObject* residual_arg, PyObject* out_arg) {
  PyObject* const no = PyLong_FromLong(kNotHandled);
  const at::Tensor *x = plain_cuda(x_arg), *y = plain_cuda(y_arg);
  if (!x || !y || x->dim() != 2) return no;
  int type;
  float eps = 0.f;
  const int dev = x->device().index();
  const int64_t M = x->size(0), N = x->size(1);
  if (!type_of(*x, &type) || dev < 0 || M <= 0 || N <= 0 || N % 8 || M > INT32_MAX || N > INT32_MAX) return no;
  const bool fp8 = scales_arg != Py_None;
  const at::Tensor* scales = fp8 ? plain_cuda(scales_arg) : nullptr;
  if (fp8 && !is_matrix(scales, M, (N + kGroup - 1) / kGroup, at::kFloat, dev)) return no;
  if (!is_matrix(y, M, N, fp8 ? at::kFloat8_e4m3fn : x->scalar_type(), dev)) return no;
  const at::Tensor *weight = nullptr, *residual = nullptr, *out = nullptr;
  if (weight_arg) {
    weight = plain_cuda(weight_arg);
    if (!weight || weight->dim() != 1 || weight->size(0) != N || weight->scalar_type() != x->scalar_type() || weight->device().index() != dev || !as_float(eps_arg, &eps)) return no;
    if (residual_arg != Py_None) {
      residual = plain_cuda(residual_arg);
      out = out_arg == Py_None ? residual : plain_cuda(out_arg);
      if (!is_matrix(residual, M, N, x->scalar_type(), dev) || !is_matrix(out, M, N, x->scalar_type(), dev)) return no;
    } else if (out_arg != Py_None) {
      return no;
    }
  }
  const void *xp = x->data_ptr(), *wp = weight ? weight->data_ptr() : nullptr, *rp = residual ? residual->data_ptr() : nullptr;
  void *yp = y->data_ptr(), *sp = scales ? scales->data_ptr() : nullptr, *op = out ? out->data_ptr() : nullptr;
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = weight ? g_rms_norm(xp, wp, rp, op, yp, sp, (int)M, (int)N, eps, type, dev, stream) : g_quantize_fp8(xp, yp, sp, (int)M, (int)N, type, dev, stream);
  Py_END_ALLOW_THREADS
  Py_DECREF(no);
  return PyLong_FromLong(rc);
}

// mul_fp8(A, B, C, sa, sb)
PyObject* mul_fp8_impl(PyObject* const* args) {
  const at::Tensor *A = plain_cuda(args[0]), *B = plain_cuda(args[1]), *C = plain_cuda(args[2]), *sa = plain_cuda(args[3]), *sb = plain_cuda(args[4]);
  int type;
  if (!A || !B || !C || !sa || !sb || A->dim() != 2 || B->dim() != 2 || !type_of(*C, &type)) return PyLong_FromLong(kNotHandled);
  const int64_t M = A->size(0), K = A->size(1), N = B->size(0), blocks = (K + kGroup - 1) / kGroup;
  const int dev = A->device().index();
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 || N % 8 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX || dev < 0 || dev >= 64 || !g_devices[dev].status ||
      A->scalar_type() != at::kFloat8_e4m3fn || !is_matrix(B, N, K, at::kFloat8_e4m3fn, dev) || !is_matrix(C, M, N, C->scalar_type(), dev) ||
      !is_matrix(sa, M, blocks, at::kFloat, dev) || !is_matrix(sb, (N + kGroup - 1) / kGroup, blocks, at::kFloat, dev))
    return PyLong_FromLong(kNotHandled);
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const auto it = scratches(kOfMulFp8).find({dev, stream});
  if (it == scratches(kOfMulFp8).end() || it->second.bytes < g_mul_fp8_scratch_bytes((int)M, (int)N, (int)K, g_devices[dev].sms)) return PyLong_FromLong(kNotHandled);
  const Scratch scratch = it->second;
  const void *a = A->data_ptr(), *b = B->data_ptr(), *ap = sa->data_ptr(), *bp = sb->data_ptr();
  void* c = C->data_ptr();
  int* status = g_devices[dev].status;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_mul_fp8(a, b, c, ap, bp, (int)M, (int)N, (int)K, type, scratch.ptr, scratch.bytes, dev, stream, status);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// A tensor of heads: four dimensions of these sizes, the values of a head next to one another, on 16-byte boundaries.
bool heads_of(const at::Tensor* t, int64_t a, int64_t b, int64_t c, int64_t d, at::ScalarType type, int dev, bool written, long long (&strides)[3]) {
  if (!t || t->dim() != 4 || t->size(0) != a || t->size(1) != b || t->size(2) != c || t->size(3) != d || t->scalar_type() != type || t->device().index() != dev ||
      t->stride(3) != 1 || reinterpret_cast<uintptr_t>(t->data_ptr()) % 16)
    return false;
  const int of = 16 / (int)t->element_size();
  for (int i = 0; i < 3; ++i) {
    strides[i] = t->size(i) == 1 ? d : t->stride(i);          // (that of a single place says nothing)
    if (strides[i] % of || (written && strides[i] == 0 && t->size(i) > 1)) return false;
  }
  return true;
}
// The bytes of a cache's powers of two.
bool scales_of(const at::Tensor* t, int64_t a, int64_t b, int64_t c, int dev, bool written, long long (&strides)[3]) {
  if (!t || t->dim() != 3 || t->size(0) != a || t->size(1) != b || t->size(2) != c || t->scalar_type() != at::kByte || t->device().index() != dev) return false;
  for (int i = 0; i < 3; ++i) {
    strides[i] = t->size(i) == 1 ? 1 : t->stride(i);
    if (written && strides[i] == 0 && t->size(i) > 1) return false;
  }
  return true;
}
// Ints of `dims` dimensions whose rows are contiguous.
bool ints_of(const at::Tensor* t, int64_t rows, int dev, int dims = 1) {
  return t && t->dim() == dims && t->size(0) == rows && t->scalar_type() == at::kInt && t->device().index() == dev && (t->size(dims - 1) <= 1 || t->stride(dims - 1) == 1);
}
bool pages_of(const at::Tensor& cache, const at::Tensor& table) {
  return cache.dim() == 4 && table.dim() == 2 && cache.size(0) > 0 && cache.size(1) > 0 && table.size(1) > 0 && cache.size(0) <= INT32_MAX && cache.size(1) <= INT32_MAX && table.size(1) <= INT32_MAX;
}

// q, k, v, k_cache, v_cache, page_table, lengths, tree, out and the scale -> the arguments of the C ABI; false: not handled
bool tree_args_of(const at::Tensor* const (&t)[9], PyObject* scale, bool fp8, fp6m_tree_attention_args* a) {
  const at::Tensor &q = *t[0], &k = *t[1], &k_cache = *t[3], &table = *t[5], &lengths = *t[6], &tree = *t[7];
  if (q.dim() != 4 || k.dim() != 4 || !pages_of(k_cache, table) || lengths.dim() != 1 || !type_of(q, &a->type)) return false;
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), G = k.size(2), pages = k_cache.size(0), page_size = k_cache.size(1), most = table.size(1);
  const int dev = q.device().index();
  const at::ScalarType type = q.scalar_type(), cache_type = fp8 ? at::kFloat8_e4m3fn : type;
  if (B <= 0 || T <= 0 || H <= 0 || T > 64 || (D != 64 && D != 128) || G <= 0 || H % G || dev < 0 || dev >= 64 || !g_devices[dev].status || B > INT32_MAX || H > INT32_MAX) return false;
  if (!heads_of(t[0], B, T, H, D, type, dev, false, a->q_stride) || !heads_of(t[1], B, T, G, D, type, dev, false, a->k_stride) ||
      !heads_of(t[2], B, T, G, D, type, dev, false, a->v_stride) || !heads_of(t[3], pages, page_size, G, D, cache_type, dev, false, a->k_cache_stride) ||
      !heads_of(t[4], pages, page_size, G, D, cache_type, dev, false, a->v_cache_stride) || !heads_of(t[8], B, T, H, D, type, dev, true, a->out_stride))
    return false;
  const bool own_masks = tree.dim() == 2;
  if (table.scalar_type() != at::kInt || table.size(0) != B || table.stride(1) != 1 || table.device().index() != dev || lengths.scalar_type() != at::kInt || lengths.size(0) != B ||
      !lengths.is_contiguous() || lengths.device().index() != dev || tree.scalar_type() != at::kLong || tree.device().index() != dev || (!own_masks && tree.dim() != 1) ||
      tree.size(own_masks ? 1 : 0) != T || (own_masks && tree.size(0) != B) || tree.stride(own_masks ? 1 : 0) != 1)
    return false;
  a->scale = D == 64 ? 0.125f : 0.08838834764831845f;
  if (scale != Py_None && !as_float(scale, &a->scale)) return false;
  a->q = q.data_ptr();
  a->k = k.data_ptr();
  a->v = t[2]->data_ptr();
  a->out = t[8]->data_ptr();
  a->k_cache = k_cache.data_ptr();
  a->v_cache = t[4]->data_ptr();
  a->page_table = static_cast<const int*>(table.data_ptr());
  a->lengths = static_cast<const int*>(lengths.data_ptr());
  a->tree = static_cast<const unsigned long long*>(tree.data_ptr());
  a->page_table_stride = table.stride(0);
  a->tree_stride = own_masks ? tree.stride(0) : 0;
  a->batch = (int)B;
  a->tokens = (int)T;
  a->heads = (int)H;
  a->kv_heads = (int)G;
  a->head_dim = (int)D;
  a->pages = (int)pages;
  a->page_size = (int)page_size;
  a->max_pages = (int)most;
  return true;
}

// tree_attention(q, k, v, k_cache, v_cache, page_table, lengths, tree, out, scale); tree_attention_fp8 has (k_scales, v_scales) behind them
PyObject* tree_attention_impl(PyObject* const* args, bool fp8) {
  const at::Tensor* t[9];
  for (int i = 0; i < 9; ++i)
    if (!(t[i] = plain_strided(args[i]))) return PyLong_FromLong(kNotHandled);
  fp6m_tree_attention_args a;
  if (!tree_args_of(t, args[9], fp8, &a)) return PyLong_FromLong(kNotHandled);
  const int dev = t[0]->device().index();
  fp6m_cache_scales s;
  if (fp8) {
    const at::Tensor *ks = plain_strided(args[10]), *vs = plain_strided(args[11]);
    if (!scales_of(ks, a.pages, a.page_size, a.kv_heads, dev, false, s.k_scales_stride) || !scales_of(vs, a.pages, a.page_size, a.kv_heads, dev, false, s.v_scales_stride)) return PyLong_FromLong(kNotHandled);
    s.k_scales = ks->data_ptr();
    s.v_scales = vs->data_ptr();
  }
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const int owner = fp8 ? kOfTreeAttentionFp8 : kOfTreeAttention;
  const auto it = scratches(owner).find({dev, stream});
  if (it == scratches(owner).end() || it->second.bytes < (fp8 ? g_tree_attention_fp8_scratch_bytes : g_tree_attention_scratch_bytes)(g_devices[dev].sms)) return PyLong_FromLong(kNotHandled);
  const Scratch scratch = it->second;
  int* status = g_devices[dev].status;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fp8 ? g_tree_attention_fp8(&a, &s, scratch.ptr, scratch.bytes, dev, stream, status) : g_tree_attention(&a, scratch.ptr, scratch.bytes, dev, stream, status);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// write_cache_fp8(k, v, k_cache, v_cache, k_scales, v_scales, page_table, lengths, tokens, counts); read_cache_fp8 has (starts) in place of the last two
PyObject* cache_impl(PyObject* const* args, bool write) {
  const at::Tensor* t[8];
  for (int i = 0; i < 8; ++i)
    if (!(t[i] = plain_strided(args[i]))) return PyLong_FromLong(kNotHandled);
  const at::Tensor &k = *t[0], &k_cache = *t[2], &table = *t[6];
  fp6m_cache_fp8_args a = {};
  fp6m_cache_scales s;
  if (k.dim() != 4 || !pages_of(k_cache, table) || !type_of(k, &a.type)) return PyLong_FromLong(kNotHandled);
  const int64_t B = k.size(0), T = k.size(1), G = k.size(2), D = k.size(3), pages = k_cache.size(0), page_size = k_cache.size(1);
  const int dev = k.device().index();
  const at::ScalarType type = k.scalar_type();
  if (B <= 0 || T <= 0 || G <= 0 || (D != 64 && D != 128) || dev < 0 || dev >= 64 || !g_devices[dev].status || B > INT32_MAX || T > INT32_MAX || G > INT32_MAX) return PyLong_FromLong(kNotHandled);
  if (!heads_of(t[0], B, T, G, D, type, dev, !write, a.k_stride) || !heads_of(t[1], B, T, G, D, type, dev, !write, a.v_stride) ||
      !heads_of(t[2], pages, page_size, G, D, at::kFloat8_e4m3fn, dev, write, a.k_cache_stride) || !heads_of(t[3], pages, page_size, G, D, at::kFloat8_e4m3fn, dev, write, a.v_cache_stride) ||
      !scales_of(t[4], pages, page_size, G, dev, write, s.k_scales_stride) || !scales_of(t[5], pages, page_size, G, dev, write, s.v_scales_stride) || !ints_of(t[6], B, dev, 2) || !ints_of(t[7], B, dev))
    return PyLong_FromLong(kNotHandled);
  a.entries = (int)T;
  for (int i = 8; i < (write ? 10 : 9); ++i) {
    if (args[i] == Py_None) continue;
    const at::Tensor* list = plain_strided(args[i]);
    const bool tokens = write && i == 8;
    if (!ints_of(list, B, dev, tokens ? 2 : 1)) return PyLong_FromLong(kNotHandled);
    const int* ptr = static_cast<const int*>(list->data_ptr());
    if (tokens) {
      if (list->size(1) <= 0 || list->size(1) > INT32_MAX) return PyLong_FromLong(kNotHandled);
      a.list = ptr;
      a.entries = (int)list->size(1);
      a.list_stride = list->stride(0);
    } else {
      (write ? a.counts : a.starts) = ptr;
    }
  }
  a.k = k.data_ptr();
  a.v = t[1]->data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = t[3]->data_ptr();
  s.k_scales = t[4]->data_ptr();
  s.v_scales = t[5]->data_ptr();
  a.page_table = static_cast<const int*>(table.data_ptr());
  a.lengths = static_cast<const int*>(t[7]->data_ptr());
  a.page_table_stride = table.stride(0);
  a.batch = (int)B;
  a.tokens = (int)T;
  a.kv_heads = (int)G;
  a.head_dim = (int)D;
  a.pages = (int)pages;
  a.page_size = (int)page_size;
  a.max_pages = (int)table.size(1);
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  int* status = g_devices[dev].status;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = (write ? g_write_cache_fp8 : g_read_cache_fp8)(&a, &s, dev, stream, status);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// verify_drafts(target, draft, drafted, tree, uniforms, accepted, counts, next_tokens)
PyObject* verify_drafts_impl(PyObject* const* args) {
  const at::Tensor* target = plain_strided(args[0]);
  const bool has_draft = args[1] != Py_None;
  const at::Tensor* draft = has_draft ? plain_strided(args[1]) : target;
  const at::Tensor *drafted = plain_cuda(args[2]), *tree = plain_strided(args[3]), *uniforms = plain_cuda(args[4]), *accepted = plain_cuda(args[5]), *counts = plain_cuda(args[6]), *next = plain_cuda(args[7]);
  if (!target || !draft || !drafted || !tree || !uniforms || !accepted || !counts || !next || target->dim() != 3 || draft->dim() != 3) return PyLong_FromLong(kNotHandled);
  fp6m_verify_drafts_args a;
  if (target->scalar_type() == at::kFloat) a.type = FP6M_TYPE_F32;
  else if (!type_of(*target, &a.type)) return PyLong_FromLong(kNotHandled);
  const int64_t B = target->size(0), T = target->size(1), V = target->size(2);
  const int dev = target->device().index();
  if (B <= 0 || T <= 0 || T > 64 || V <= 0 || B > INT32_MAX || V > INT32_MAX || dev < 0) return PyLong_FromLong(kNotHandled);
  for (const at::Tensor* t : {target, draft})
    if (t->size(0) != B || t->size(1) != T || t->size(2) != V || (V > 1 && t->stride(2) != 1) || t->scalar_type() != target->scalar_type() || t->device().index() != dev) return PyLong_FromLong(kNotHandled);
  const bool own_masks = tree->dim() == 2;
  if (!is_matrix(drafted, B, T, at::kLong, dev) || !is_matrix(uniforms, B, T, at::kFloat, dev) || !is_matrix(accepted, B, T, at::kInt, dev) || counts->dim() != 1 || counts->size(0) != B ||
      counts->scalar_type() != at::kInt || counts->device().index() != dev || next->dim() != 1 || next->size(0) != B || next->scalar_type() != at::kLong || next->device().index() != dev ||
      tree->scalar_type() != at::kLong || tree->device().index() != dev || (!own_masks && tree->dim() != 1) || tree->size(own_masks ? 1 : 0) != T || (own_masks && tree->size(0) != B) ||
      (T > 1 && tree->stride(own_masks ? 1 : 0) != 1))
    return PyLong_FromLong(kNotHandled);
  a.target = target->data_ptr();
  a.draft = has_draft ? draft->data_ptr() : nullptr;
  a.drafted = static_cast<const long long*>(drafted->data_ptr());
  a.tree = static_cast<const unsigned long long*>(tree->data_ptr());
  a.uniforms = static_cast<const float*>(uniforms->data_ptr());
  a.accepted = static_cast<int*>(accepted->data_ptr());
  a.counts = static_cast<int*>(counts->data_ptr());
  a.next_tokens = static_cast<long long*>(next->data_ptr());
  for (int i = 0; i < 2; ++i) {
    a.target_stride[i] = target->stride(i);
    a.draft_stride[i] = draft->stride(i);
  }
  a.tree_stride = own_masks ? tree->stride(0) : 0;
  a.batch = (int)B;
  a.tokens = (int)T;
  a.vocab = (int)V;
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_verify_drafts(&a, dev, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// what a call returns, with torch's exceptions as Python's
template <class F>
PyObject* guarded(const char* name, Py_ssize_t nargs, Py_ssize_t expected, F&& call) {
  if (nargs != expected) {
    PyErr_Format(PyExc_TypeError, "%s: %d arguments", name, (int)expected);
    return nullptr;
  }
  try {
    return call();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("rms_norm", nargs, 7, [&] { return rows_impl(args[0], args[1], args[2], args[3], args[4], args[5], args[6]); });
}
PyObject* py_quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("quantize_fp8", nargs, 3, [&] { return rows_impl(args[0], nullptr, args[1], nullptr, args[2], Py_None, Py_None); });
}
PyObject* py_mul_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("mul_fp8", nargs, 5, [&] { return mul_fp8_impl(args); });
}
PyObject* py_tree_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("tree_attention", nargs, 10, [&] { return tree_attention_impl(args, false); });
}
PyObject* py_tree_attention_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("tree_attention_fp8", nargs, 12, [&] { return tree_attention_impl(args, true); });
}
PyObject* py_write_cache_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("write_cache_fp8", nargs, 10, [&] { return cache_impl(args, true); });
}
PyObject* py_read_cache_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("read_cache_fp8", nargs, 9, [&] { return cache_impl(args, false); });
}
PyObject* py_verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("verify_drafts", nargs, 8, [&] { return verify_drafts_impl(args); });
}

PyObject* py_mul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 13) {
    PyErr_SetString(PyExc_TypeError, "mul: 13 arguments");
    return nullptr;
  }
  try {
    return mul_impl(args);
  } catch (const std::exception& e) {          // (torch's accessors report errors as exceptions)
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// bind(mul, mul_fused, scratch_bytes): addresses of the C ABI's functions
PyObject* py_bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c;
  if (!PyArg_ParseTuple(args, "KKK", &a, &b, &c)) return nullptr;
  g_mul = reinterpret_cast<MulFn>(a);
  g_mul_fused = reinterpret_cast<MulFusedFn>(b);
  g_scratch_bytes = reinterpret_cast<ScratchFn>(c);
  Py_RETURN_NONE;
}

// bind_operators(rms_norm, quantize_fp8, mul_fp8, its scratch_bytes, tree_attention, its scratch_bytes, write_cache_fp8, read_cache_fp8, tree_attention_fp8, its
// scratch_bytes, verify_drafts): likewise
PyObject* py_bind_operators(PyObject*, PyObject* args) {
  unsigned long long a[11];
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9], &a[10])) return nullptr;
  int i = 0;
  auto set = [&](auto& function) { function = reinterpret_cast<std::remove_reference_t<decltype(function)>>(a[i++]); };
  set(g_rms_norm);
  set(g_quantize_fp8);
  set(g_mul_fp8);
  set(g_mul_fp8_scratch_bytes);
  set(g_tree_attention);
  set(g_tree_attention_scratch_bytes);
  set(g_write_cache_fp8);
  set(g_read_cache_fp8);
  set(g_tree_attention_fp8);
  set(g_tree_attention_fp8_scratch_bytes);
  set(g_verify_drafts);
  Py_RETURN_NONE;
}

// set_device(dev, address of the status word, multiprocessors)
PyObject* py_set_device(PyObject*, PyObject* args) {
  int dev, sms;
  unsigned long long status;
  if (!PyArg_ParseTuple(args, "iKi", &dev, &status, &sms)) return nullptr;
  if (dev >= 0 && dev < 64) {
    g_devices[dev].status = reinterpret_cast<int*>(status);
    g_devices[dev].sms = sms;
  }
  Py_RETURN_NONE;
}

// set_scratch(dev, stream, address, bytes); the caller keeps the memory for the life of the process
PyObject* py_set_scratch(PyObject*, PyObject* args) {
  int dev;
  unsigned long long stream, ptr, bytes;
  if (!PyArg_ParseTuple(args, "iKKK", &dev, &stream, &ptr, &bytes)) return nullptr;
  try {
    scratches()[{dev, reinterpret_cast<void*>(stream)}] = {reinterpret_cast<void*>(ptr), (size_t)bytes};
  } catch (const std::bad_alloc&) {
    return PyErr_NoMemory();
  }
  Py_RETURN_NONE;
}

// set_operator_scratch(owner, dev, stream, address, bytes): likewise, of mul_fp8 (1), tree_attention (2) or tree_attention_fp8 (3)
PyObject* py_set_operator_scratch(PyObject*, PyObject* args) {
  int owner, dev;
  unsigned long long stream, ptr, bytes;
  if (!PyArg_ParseTuple(args, "iiKKK", &owner, &dev, &stream, &ptr, &bytes)) return nullptr;
  if (owner <= kOfGemms || owner >= kOwners) {
    PyErr_SetString(PyExc_ValueError, "set_operator_scratch: unknown owner");
    return nullptr;
  }
  try {
    scratches(owner)[{dev, reinterpret_cast<void*>(stream)}] = {reinterpret_cast<void*>(ptr), (size_t)bytes};
  } catch (const std::bad_alloc&) {
    return PyErr_NoMemory();
  }
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"rms_norm", (PyCFunction)(void (*)(void))py_rms_norm, METH_FASTCALL, "norm of the rows of plain CUDA tensors: C ABI status, or -1 when the call is not handled here"},
    {"quantize_fp8", (PyCFunction)(void (*)(void))py_quantize_fp8, METH_FASTCALL, "rows to E4M3, likewise"},
    {"mul_fp8", (PyCFunction)(void (*)(void))py_mul_fp8, METH_FASTCALL, "8-bit product, likewise"},
    {"tree_attention", (PyCFunction)(void (*)(void))py_tree_attention, METH_FASTCALL, "attention over a paged cache, likewise"},
    {"tree_attention_fp8", (PyCFunction)(void (*)(void))py_tree_attention_fp8, METH_FASTCALL, "attention over a cache in 8 bits, likewise"},
    {"write_cache_fp8", (PyCFunction)(void (*)(void))py_write_cache_fp8, METH_FASTCALL, "tokens into a cache in 8 bits, likewise"},
    {"read_cache_fp8", (PyCFunction)(void (*)(void))py_read_cache_fp8, METH_FASTCALL, "tokens out of it, likewise"},
    {"verify_drafts", (PyCFunction)(void (*)(void))py_verify_drafts, METH_FASTCALL, "verification of drafted tokens, likewise"},
    {"bind_operators", py_bind_operators, METH_VARARGS, "addresses of the C ABI's functions of the operators"},
    {"set_operator_scratch", py_set_operator_scratch, METH_VARARGS, "scratch of an operator on a device's stream"},
    {"mul", (PyCFunction)(void (*)(void))py_mul, METH_FASTCALL, "GEMM on plain CUDA tensors: C ABI status, or -1 when the call is not handled here"},
    {"bind", py_bind, METH_VARARGS, "addresses of the C ABI's functions"},
    {"set_device", py_set_device, METH_VARARGS, "status word and number of multiprocessors of a device"},
    {"set_scratch", py_set_scratch, METH_VARARGS, "split-K scratch of a device's stream"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_call", "host call path of mul and mul_fused", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call(void) {
  PyObject* module = PyModule_Create(&kModule);
  // the importer compares it with the torch it has: torch's accessors are inlined here
  if (module && PyModule_AddStringConstant(module, "torch_version", FP6M_TORCH_VERSION) != 0) Py_CLEAR(module);
  return module;
}
