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
  for (int i = 0; i < 3; ++i) {
    strides[i] = t->size(i) == 1 ? d : t->stride(i);          // (that of a single place says nothing)
    if (strides[i] % 8 || (written && strides[i] == 0 && t->size(i) > 1)) return false;
  }
  return true;
}

// tree_attention(q, k, v, k_cache, v_cache, page_table, lengths, tree, out, scale)
PyObject* tree_attention_impl(PyObject* const* args) {
  const at::Tensor* t[9];
  for (int i = 0; i < 9; ++i)
    if (!(t[i] = plain_strided(args[i]))) return PyLong_FromLong(kNotHandled);
  const at::Tensor &q = *t[0], &k = *t[1], &k_cache = *t[3], &table = *t[5], &lengths = *t[6], &tree = *t[7];
  fp6m_tree_attention_args a;
  if (q.dim() != 4 || k.dim() != 4 || k_cache.dim() != 4 || table.dim() != 2 || lengths.dim() != 1 || !type_of(q, &a.type)) return PyLong_FromLong(kNotHandled);
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), G = k.size(2), pages = k_cache.size(0), page_size = k_cache.size(1), most = table.size(1);
  const int dev = q.device().index();
  const at::ScalarType type = q.scalar_type();
  if (B <= 0 || T <= 0 || H <= 0 || T > 64 || (D != 64 && D != 128) || G <= 0 || H % G || pages <= 0 || page_size <= 0 || most <= 0 || dev < 0 || dev >= 64 ||
      !g_devices[dev].status || B > INT32_MAX || H > INT32_MAX || pages > INT32_MAX || page_size > INT32_MAX || most > INT32_MAX)
    return PyLong_FromLong(kNotHandled);
  if (!heads_of(t[0], B, T, H, D, type, dev, false, a.q_stride) || !heads_of(t[1], B, T, G, D, type, dev, false, a.k_stride) ||
      !heads_of(t[2], B, T, G, D, type, dev, false, a.v_stride) || !heads_of(t[3], pages, page_size, G, D, type, dev, false, a.k_cache_stride) ||
      !heads_of(t[4], pages, page_size, G, D, type, dev, false, a.v_cache_stride) || !heads_of(t[8], B, T, H, D, type, dev, true, a.out_stride))
    return PyLong_FromLong(kNotHandled);
  const bool own_masks = tree.dim() == 2;
  if (table.scalar_type() != at::kInt || table.size(0) != B || table.stride(1) != 1 || table.device().index() != dev || lengths.scalar_type() != at::kInt || lengths.size(0) != B ||
      !lengths.is_contiguous() || lengths.device().index() != dev || tree.scalar_type() != at::kLong || tree.device().index() != dev || (!own_masks && tree.dim() != 1) ||
      tree.size(own_masks ? 1 : 0) != T || (own_masks && tree.size(0) != B) || tree.stride(own_masks ? 1 : 0) != 1)
    return PyLong_FromLong(kNotHandled);
  a.scale = D == 64 ? 0.125f : 0.08838834764831845f;
  if (args[9] != Py_None && !as_float(args[9], &a.scale)) return PyLong_FromLong(kNotHandled);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = t[2]->data_ptr();
  a.out = t[8]->data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = t[4]->data_ptr();
  a.page_table = static_cast<const int*>(table.data_ptr());
  a.lengths = static_cast<const int*>(lengths.data_ptr());
  a.tree = static_cast<const unsigned long long*>(tree.data_ptr());
  a.page_table_stride = table.stride(0);
  a.tree_stride = own_masks ? tree.stride(0) : 0;
  a.batch = (int)B;
  a.tokens = (int)T;
  a.heads = (int)H;
  a.kv_heads = (int)G;
  a.head_dim = (int)D;
  a.pages = (int)pages;
  a.page_size = (int)page_size;
  a.max_pages = (int)most;
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  const auto it = scratches(kOfTreeAttention).find({dev, stream});
  if (it == scratches(kOfTreeAttention).end() || it->second.bytes < g_tree_attention_scratch_bytes(g_devices[dev].sms)) return PyLong_FromLong(kNotHandled);
  const Scratch scratch = it->second;
  int* status = g_devices[dev].status;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_tree_attention(&a, scratch.ptr, scratch.bytes, dev, stream, status);
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
  return guarded("tree_attention", nargs, 10, [&] { return tree_attention_impl(args); });
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

// bind_operators(rms_norm, quantize_fp8, mul_fp8, its scratch_bytes, tree_attention, its scratch_bytes): likewise
PyObject* py_bind_operators(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d, e, f;
  if (!PyArg_ParseTuple(args, "KKKKKK", &a, &b, &c, &d, &e, &f)) return nullptr;
  g_rms_norm = reinterpret_cast<decltype(g_rms_norm)>(a);
  g_quantize_fp8 = reinterpret_cast<decltype(g_quantize_fp8)>(b);
  g_mul_fp8 = reinterpret_cast<decltype(g_mul_fp8)>(c);
  g_mul_fp8_scratch_bytes = reinterpret_cast<decltype(g_mul_fp8_scratch_bytes)>(d);
  g_tree_attention = reinterpret_cast<decltype(g_tree_attention)>(e);
  g_tree_attention_scratch_bytes = reinterpret_cast<decltype(g_tree_attention_scratch_bytes)>(f);
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
