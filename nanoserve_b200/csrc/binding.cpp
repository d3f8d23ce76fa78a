// The host side of ops.Kernels.w4_linear and w4_quantize, and of the operators of batched serving, as one native call each.
// Through ctypes an eager one-token call spent more time in Python (argument conversion, torch.empty with keywords, the tensors'
// properties) than its launch takes; here the same steps run on the tensors' C++ objects (512 x 3584 at one token 8.6 -> 4.8 us a
// call).
//
// w4_linear(fn, x, Wq, S, group, flags, out): `fn` is the address of b2_w4_linear in whatever library the caller has loaded.
// w4_quantize(fn, W, group): likewise of ns_w4_quantize.  paged_kv_append, paged_attention, shared_prefix_attention and sample
// take the arguments of their methods in order, behind the addresses of their entry points (for the two attentions that of the
// workspace's size too), and check what the methods check.  They take exactly torch.Tensor (or Parameter) arguments on a CUDA
// device, x and W matrices; for anything else -- a subclass, a tensor on the host, an active dispatch or function mode, other
// argument types -- they return NotImplemented before they have done anything, and the caller takes its own path, which then
// answers or refuses as ever.
#include <Python.h>

#include <cmath>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/nanoserve_b200.h"

namespace {

using LinearFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int, int, void*);
using QuantizeFn = int (*)(const void*, void*, void*, int, int, int, void*);

bool plain(PyObject* o) { return THPVariable_CheckExact(o); }

bool modes_active() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
         c10::impl::tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

bool as_int(PyObject* o, int* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow || v < INT32_MIN || v > INT32_MAX) return false;
  *out = (int)v;
  return true;
}

PyObject* w4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int group = 0, flags = 0;
  if (n != 7 || !PyLong_CheckExact(a[0]) || !plain(a[1]) || !plain(a[2]) || !plain(a[3]) || !as_int(a[4], &group) ||
      !as_int(a[5], &flags) || !(a[6] == Py_None || plain(a[6])) || modes_active())
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor& x0 = THPVariable_Unpack(a[1]);
  const at::Tensor& wq = THPVariable_Unpack(a[2]);
  const at::Tensor& s = THPVariable_Unpack(a[3]);
  if (!x0.is_cuda() || !wq.is_cuda() || !s.is_cuda() || x0.dim() != 2 || wq.dim() < 1 || x0.size(0) > INT32_MAX ||
      x0.size(1) > INT32_MAX || wq.size(0) > INT32_MAX || !x0.has_storage() || !wq.has_storage() || !s.has_storage())
    Py_RETURN_NOTIMPLEMENTED;
  if (a[6] != Py_None && (!THPVariable_Unpack(a[6]).is_cuda() || !THPVariable_Unpack(a[6]).has_storage()))
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor x = x0.is_contiguous() ? x0 : x0.contiguous();
  const int M = (int)x.size(0), K = (int)x.size(1), N = (int)wq.size(0);
  const at::Tensor y = a[6] != Py_None ? THPVariable_Unpack(a[6])
                                       : at::empty({M, N}, at::TensorOptions().dtype(at::kBFloat16).device(x.device()));
  const auto fn = reinterpret_cast<LinearFn>(PyLong_AsVoidPtr(a[0]));
  const void *xp = x.const_data_ptr(), *wp = wq.const_data_ptr(), *sp = s.const_data_ptr();
  void* const yp = y.mutable_data_ptr();
  void* const stream = c10::cuda::getCurrentCUDAStream().stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(xp, wp, sp, yp, M, N, K, group, flags, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_Format(PyExc_RuntimeError, "ns_w4_linear failed with code %d", rc);
    return nullptr;
  }
  if (a[6] != Py_None) {
    Py_INCREF(a[6]);
    return a[6];
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* w4_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int group = 0;
  if (n != 3 || !PyLong_CheckExact(a[0]) || !plain(a[1]) || !as_int(a[2], &group) || group < 1 || modes_active())
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor& w0 = THPVariable_Unpack(a[1]);
  if (!w0.is_cuda() || w0.dim() != 2 || w0.size(0) > INT32_MAX || w0.size(1) > INT32_MAX || !w0.has_storage())
    Py_RETURN_NOTIMPLEMENTED;
  const int64_t N = w0.size(0), K = w0.size(1);
  const at::Tensor wq = at::empty({N, K / 8}, at::TensorOptions().dtype(at::kInt).device(w0.device()));
  const at::Tensor s = at::empty({N, K / group}, at::TensorOptions().dtype(at::kBFloat16).device(w0.device()));
  const at::Tensor w = w0.is_contiguous() ? w0 : w0.contiguous();
  const auto fn = reinterpret_cast<QuantizeFn>(PyLong_AsVoidPtr(a[0]));
  const void* const wp = w.const_data_ptr();
  void *const qp = wq.mutable_data_ptr(), *const sp = s.mutable_data_ptr();
  void* const stream = c10::cuda::getCurrentCUDAStream().stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(wp, qp, sp, (int)N, (int)K, group, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_Format(PyExc_RuntimeError, "ns_w4_quantize failed with code %d", rc);
    return nullptr;
  }
  PyObject* const q = THPVariable_Wrap(wq);
  PyObject* const t = q ? THPVariable_Wrap(s) : nullptr;
  if (!t) {
    Py_XDECREF(q);
    return nullptr;
  }
  PyObject* const both = PyTuple_Pack(2, q, t);
  Py_DECREF(q);
  Py_DECREF(t);
  return both;
  END_HANDLE_TH_ERRORS
}

// ---- several sequences: a paged cache, attention over it, sampling

const at::Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }
bool on_device(PyObject* o) { return plain(o) && tensor(o).is_cuda(); }  // (asked before the current device: there may be none)
// A plain tensor on the current device.
bool here(PyObject* o, int dev) {
  if (!plain(o)) return false;
  const at::Tensor& t = tensor(o);
  return t.is_cuda() && t.get_device() == dev && t.has_storage();
}
bool here_or_none(PyObject* o, int dev) { return o == Py_None || here(o, dev); }
bool is_vector(const at::Tensor& t, at::ScalarType type, int64_t n) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && (n < 2 || t.stride(0) == 1);
}
bool is_rows(const at::Tensor& t, int64_t rows, int64_t width) {
  return t.scalar_type() == at::kBFloat16 && t.dim() == 2 && (rows < 0 || t.size(0) == rows) && t.size(0) <= INT32_MAX &&
         t.size(1) == width && t.stride(1) == 1;
}
const void* address(PyObject* o) { return o == Py_None ? nullptr : tensor(o).const_data_ptr(); }

// k, v, block_table, seq_lens, [n_heads,] n_kv_heads, head_dim as the methods take them.
bool paged(PyObject* const* a, int n_heads, int Hk, int D, int dev, b2_paged_cache* c) {
  if (!here(a[0], dev) || !here(a[1], dev) || !here(a[2], dev) || !here(a[3], dev) || n_heads < 1 || Hk < 1 || D < 1) return false;
  const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &table = tensor(a[2]), &lens = tensor(a[3]);
  if (k.dim() != 4 || v.dim() != 4 || k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16 ||
      k.sizes() != v.sizes() || k.strides() != v.strides() || k.size(1) != Hk || k.size(3) != D || k.stride(3) != 1 ||
      k.size(0) > INT32_MAX || k.size(2) > INT32_MAX)
    return false;
  if (lens.dim() != 1 || !is_vector(lens, at::kInt, lens.size(0)) || lens.size(0) > INT32_MAX || table.dim() != 2 ||
      table.scalar_type() != at::kInt || table.size(0) != lens.size(0) || table.size(1) > INT32_MAX ||
      (table.stride(1) != 1 && table.size(1) != 1))
    return false;
  c->k = const_cast<void*>(k.const_data_ptr());
  c->v = const_cast<void*>(v.const_data_ptr());
  c->page_stride = k.stride(0);
  c->head_stride = k.stride(1);
  c->token_stride = k.stride(2);
  c->n_pages = (int)k.size(0);
  c->page_size = (int)k.size(2);
  c->n_kv_heads = Hk;
  c->head_dim = D;
  c->block_table = table.const_data_ptr();
  c->table_stride = table.stride(0);
  c->table_width = (int)table.size(1);
  c->n_seqs = (int)lens.size(0);
  c->seq_lens = lens.const_data_ptr();
  return true;
}
bool cu_fits(PyObject* cu, int64_t rows, int n_seqs) {
  return cu == Py_None ? rows == n_seqs : is_vector(tensor(cu), at::kInt, (int64_t)n_seqs + 1);
}
PyObject* answer(int rc, const char* name, PyObject* given, const at::Tensor& out) {
  if (rc != 0) return PyErr_Format(PyExc_RuntimeError, "%s failed with code %d", name, rc);
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(out);
}
at::Tensor room(int64_t rows, int64_t width, at::ScalarType type, int dev) {
  const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, dev);
  return width < 0 ? at::empty({rows}, options) : at::empty({rows, width}, options);
}
bool as_scale(PyObject* o, int D, float* out) {
  if (o != Py_None && !PyFloat_CheckExact(o)) return false;
  *out = o == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)PyFloat_AS_DOUBLE(o);
  return true;
}

// fn, qkv, bias, inv_freq, cache_k, cache_v, block_table, seq_lens, n_heads, n_kv_heads, head_dim, cu_tokens, q_out
PyObject* paged_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int Hq = 0, Hk = 0, D = 0;
  b2_paged_cache c;
  if (n != 13 || !PyLong_CheckExact(a[0]) || !as_int(a[8], &Hq) || !as_int(a[9], &Hk) || !as_int(a[10], &D) || !on_device(a[1]) || modes_active())
    Py_RETURN_NOTIMPLEMENTED;
  const int dev = c10::cuda::current_device();
  if (!here(a[1], dev) || !here_or_none(a[2], dev) || !here(a[3], dev) || !paged(a + 4, Hq, Hk, D, dev, &c) ||
      !here_or_none(a[11], dev) || !here_or_none(a[12], dev))
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor& x = tensor(a[1]);
  const int64_t width = ((int64_t)Hq + 2 * (int64_t)Hk) * D;
  if (!is_rows(x, -1, width) || x.size(0) < 1 || !cu_fits(a[11], x.size(0), c.n_seqs) ||
      !is_vector(tensor(a[3]), at::kFloat, D / 2) || (a[2] != Py_None && !is_vector(tensor(a[2]), at::kBFloat16, width)) ||
      (a[12] != Py_None && !is_rows(tensor(a[12]), x.size(0), (int64_t)Hq * D)))
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor q = a[12] != Py_None ? tensor(a[12]) : room(x.size(0), (int64_t)Hq * D, at::kBFloat16, dev);
  const auto fn = reinterpret_cast<decltype(&b2_paged_kv_append)>(PyLong_AsVoidPtr(a[0]));
  const void *xp = x.const_data_ptr(), *bias = address(a[2]), *inv = address(a[3]), *cu = address(a[11]);
  void *const qp = q.mutable_data_ptr(), *const stream = c10::cuda::getCurrentCUDAStream().stream();
  const int64_t xs = x.stride(0), qs = q.stride(0), T = x.size(0);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(xp, xs, bias, inv, qp, qs, &c, cu, (int)T, Hq, stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "b2_paged_kv_append", a[12], q);
  END_HANDLE_TH_ERRORS
}

// fn, size, q, cache_k, cache_v, block_table, seq_lens, n_heads, n_kv_heads, head_dim, cu_tokens, max_tokens, window, sinks,
// scale, out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int Hq = 0, Hk = 0, D = 0, most = 0, window = 0, sinks = 0;
  float scale = 0.f;
  b2_paged_cache c;
  if (n != 16 || !PyLong_CheckExact(a[0]) || !PyLong_CheckExact(a[1]) || !as_int(a[7], &Hq) || !as_int(a[8], &Hk) ||
      !as_int(a[9], &D) || !(a[11] == Py_None || as_int(a[11], &most)) || !as_int(a[12], &window) || !as_int(a[13], &sinks) ||
      D < 1 || !as_scale(a[14], D, &scale) || !on_device(a[2]) || modes_active())
    Py_RETURN_NOTIMPLEMENTED;
  const int dev = c10::cuda::current_device();
  if (!here(a[2], dev) || !paged(a + 3, Hq, Hk, D, dev, &c) || !here_or_none(a[10], dev) || !here_or_none(a[15], dev))
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor& q = tensor(a[2]);
  const int64_t width = (int64_t)Hq * D;
  if (!is_rows(q, -1, width) || q.size(0) < 1 || !cu_fits(a[10], q.size(0), c.n_seqs) ||
      (a[15] != Py_None && !is_rows(tensor(a[15]), q.size(0), width)))
    Py_RETURN_NOTIMPLEMENTED;
  const int T = (int)q.size(0);
  if (a[11] == Py_None) most = a[10] == Py_None ? 1 : T;
  const auto fn = reinterpret_cast<decltype(&b2_paged_attention)>(PyLong_AsVoidPtr(a[0]));
  const auto size = reinterpret_cast<decltype(&b2_paged_attention_workspace_bytes)>(PyLong_AsVoidPtr(a[1]));
  const at::Tensor out = a[15] != Py_None ? tensor(a[15]) : room(T, width, at::kBFloat16, dev);
  const size_t bytes = size(T, c.n_seqs, most, Hq, Hk, D);
  const at::Tensor ws = room((int64_t)bytes, -1, at::kByte, dev);
  const void *qp = q.const_data_ptr(), *cu = address(a[10]);
  void *const op = out.mutable_data_ptr(), *const wp = ws.mutable_data_ptr();
  void* const stream = c10::cuda::getCurrentCUDAStream().stream();
  const int64_t qs = q.stride(0), os = out.stride(0);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(qp, qs, &c, cu, T, most, Hq, window, sinks, scale, op, os, wp, bytes, stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "b2_paged_attention", a[15], out);
  END_HANDLE_TH_ERRORS
}

// fn, size, q, cache_k, cache_v, prefix_table, prefix_len, block_table, seq_lens, n_heads, n_kv_heads, head_dim, scale, out
PyObject* shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int Hq = 0, Hk = 0, D = 0;
  float scale = 0.f;
  b2_paged_cache c;
  if (n != 14 || !PyLong_CheckExact(a[0]) || !PyLong_CheckExact(a[1]) || !as_int(a[9], &Hq) || !as_int(a[10], &Hk) ||
      !as_int(a[11], &D) || D < 1 || !as_scale(a[12], D, &scale) || !on_device(a[2]) || modes_active())
    Py_RETURN_NOTIMPLEMENTED;
  const int dev = c10::cuda::current_device();
  PyObject* const cache[4] = {a[3], a[4], a[7], a[8]};
  if (!here(a[2], dev) || !paged(cache, Hq, Hk, D, dev, &c) || !here(a[5], dev) || !here(a[6], dev) || !here_or_none(a[13], dev))
    Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor &q = tensor(a[2]), &table = tensor(a[5]), &len = tensor(a[6]);
  const int64_t width = (int64_t)Hq * D;
  if (c.n_seqs < 1 || !is_rows(q, c.n_seqs, width) || table.dim() != 1 || table.size(0) > INT32_MAX || !is_vector(table, at::kInt, table.size(0)) ||
      len.scalar_type() != at::kInt || len.numel() != 1 || (a[13] != Py_None && !is_rows(tensor(a[13]), c.n_seqs, width)))
    Py_RETURN_NOTIMPLEMENTED;
  const auto fn = reinterpret_cast<decltype(&b2_shared_prefix_attention)>(PyLong_AsVoidPtr(a[0]));
  const auto size = reinterpret_cast<decltype(&b2_shared_prefix_workspace_bytes)>(PyLong_AsVoidPtr(a[1]));
  const at::Tensor out = a[13] != Py_None ? tensor(a[13]) : room(c.n_seqs, width, at::kBFloat16, dev);
  const size_t bytes = size(c.n_seqs, Hq, Hk, D);
  const at::Tensor ws = room((int64_t)bytes, -1, at::kByte, dev);
  const void *qp = q.const_data_ptr(), *tp = table.const_data_ptr(), *lp = len.const_data_ptr();
  void *const op = out.mutable_data_ptr(), *const wp = ws.mutable_data_ptr();
  void* const stream = c10::cuda::getCurrentCUDAStream().stream();
  const int64_t qs = q.stride(0), os = out.stride(0);
  const int pages = (int)table.size(0);
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(qp, qs, &c, tp, pages, lp, Hq, scale, op, os, wp, bytes, stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "b2_shared_prefix_attention", a[13], out);
  END_HANDLE_TH_ERRORS
}

// fn, logits, u, temperature, top_k, top_p, min_p, out
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !PyLong_CheckExact(a[0]) || !on_device(a[1]) || modes_active()) Py_RETURN_NOTIMPLEMENTED;
  const int dev = c10::cuda::current_device();
  if (!here(a[1], dev) || !here(a[2], dev) || !here_or_none(a[7], dev)) Py_RETURN_NOTIMPLEMENTED;
  const at::Tensor &x = tensor(a[1]), &u = tensor(a[2]);
  if (x.dim() != 2 || (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kFloat) || x.size(0) < 1 ||
      x.size(0) > INT32_MAX || x.size(1) > INT32_MAX || (x.stride(1) != 1 && x.size(1) != 1) ||
      !is_vector(u, at::kFloat, x.size(0)) || (a[7] != Py_None && !is_vector(tensor(a[7]), at::kLong, x.size(0))))
    Py_RETURN_NOTIMPLEMENTED;
  const void* arrays[4];
  float values[4] = {1.f, 0.f, 1.f, 0.f};
  int top_k = 0;
  for (int i = 0; i < 4; ++i) {
    PyObject* const o = a[3 + i];
    arrays[i] = nullptr;
    if (here(o, dev)) {
      if (!is_vector(tensor(o), i == 1 ? at::kInt : at::kFloat, x.size(0))) Py_RETURN_NOTIMPLEMENTED;
      arrays[i] = tensor(o).const_data_ptr();
    } else if (i == 1) {
      if (!as_int(o, &top_k)) Py_RETURN_NOTIMPLEMENTED;
    } else if (PyFloat_CheckExact(o)) {
      values[i] = (float)PyFloat_AS_DOUBLE(o);
    } else {
      Py_RETURN_NOTIMPLEMENTED;
    }
  }
  const at::Tensor out = a[7] != Py_None ? tensor(a[7]) : room(x.size(0), -1, at::kLong, dev);
  const auto fn = reinterpret_cast<decltype(&b2_sample)>(PyLong_AsVoidPtr(a[0]));
  const void *xp = x.const_data_ptr(), *up = u.const_data_ptr();
  void *const op = out.mutable_data_ptr(), *const stream = c10::cuda::getCurrentCUDAStream().stream();
  const int64_t stride = x.stride(0), B = x.size(0), V = x.size(1);
  const int fp32 = x.scalar_type() == at::kFloat;
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(xp, stride, fp32, (int)B, (int)V, up, arrays[0], arrays[1], arrays[2], arrays[3], values[0], top_k, values[2], values[3],
          op, stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "b2_sample", a[7], out);
  END_HANDLE_TH_ERRORS
}

#define B2_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {B2_FAST(w4_linear), B2_FAST(w4_quantize), B2_FAST(paged_kv_append), B2_FAST(paged_attention),
                          B2_FAST(shared_prefix_attention), B2_FAST(sample), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "nanoserve_call", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit_nanoserve_call(void) { return PyModule_Create(&kModule); }
