// The host side of compressai_b200.attention as a CPython module: argument checks, output and
// workspace allocation, and the call of the C-ABI on the current stream.
//
// One token's rotary is 2 us of GPU time and a decode step's attention 8, while the same checks in
// Python with a ctypes call of 20 to 30 arguments took 15 to 21 us (B200 host); this module takes
// the place of both. The entry points are the library's, by the addresses that _lib has bound.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <stdexcept>
#include <string>

#include "vq2_b200.h"

namespace {

decltype(&vq2_rotary) f_rotary;
decltype(&vq2_cache_write) f_write;
decltype(&vq2_cache_read) f_read;
decltype(&vq2_paged_attention) f_attention;
decltype(&vq2_paged_attention_workspace) f_workspace;
PyObject *check_status, *out_of_memory;   // _lib.check(status, name); torch.OutOfMemoryError

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Raised {};   // a Python exception is set

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused(s.str());
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
int truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v;
}

int code(at::ScalarType t) {
  return t == at::kHalf ? VQ2_F16 : t == at::kBFloat16 ? VQ2_BF16 : t == at::kChar ? VQ2_I8 : -1;
}

void on_cuda(const at::Tensor& t) {
  if (!t.is_cuda())
    refuse("compressai_b200 kernels take CUDA tensors only (no CPU fallback); got a tensor on ", t.device());
}

// [tokens, heads, head_size] in fp16 or bf16; the last dimension made contiguous.
at::Tensor rows(const at::Tensor& x, const char* name, const at::Tensor* like = nullptr) {
  on_cuda(x);
  const int c = code(x.scalar_type());
  if (x.dim() != 3 || (c != VQ2_F16 && c != VQ2_BF16))
    refuse(name, " must be [tokens, heads, head_size] in fp16 or bf16; got ", x.sizes(), " ", x.scalar_type());
  if (like && (x.scalar_type() != like->scalar_type() || x.size(0) != like->size(0) || x.size(2) != like->size(2) ||
               x.device() != like->device()))
    refuse(name, " ", x.sizes(), " ", x.scalar_type(), " on ", x.device(), " does not go with ", like->sizes(), " ",
           like->scalar_type(), " on ", like->device());
  return x.stride(2) == 1 || x.size(2) == 1 ? x : x.contiguous();
}

const int32_t* ints(const at::Tensor& x, const char* name, int64_t n, c10::Device dev) {
  if (x.scalar_type() != at::kInt || x.dim() != 1 || x.size(0) != n || x.device() != dev || !x.is_contiguous())
    refuse(name, " must be a contiguous int32 tensor of ", n, " on ", dev, "; got ", x.scalar_type(), " ", x.sizes(), " on ",
           x.device());
  return static_cast<const int32_t*>(x.const_data_ptr());
}

struct Pools {
  void *k, *v;
  float *ks = nullptr, *vs = nullptr;
  int kind;
  int64_t pages, heads, page, d, stride, cols, seqs;
  const int32_t* table;
};

// The cache's arguments; dtype < 0, heads < 0, d < 0: not known.
Pools pools(PyObject* const* a, int dtype, int64_t heads, int64_t d, c10::Device dev) {  // k, v, table, k_scale, v_scale
  const at::Tensor &k = tensor(a[0], "k_pages"), &v = tensor(a[1], "v_pages"), &table = tensor(a[2], "table");
  const at::Tensor *ks = maybe(a[3], "k_scale"), *vs = maybe(a[4], "v_scale");
  Pools p;
  p.kind = code(k.scalar_type());
  if (p.kind < 0 || v.scalar_type() != k.scalar_type())
    refuse("pools hold fp16, bf16 or int8, both the same; got ", k.scalar_type(), " and ", v.scalar_type());
  if (k.dim() != 4 || k.sizes() != v.sizes() || !k.is_contiguous() || !v.is_contiguous())
    refuse("pools must be contiguous [pages, kv_heads, page_size, head_size], k and v alike; got ", k.sizes(), " and ", v.sizes());
  if (k.device() != dev || v.device() != dev) refuse("pools on ", k.device(), " and ", v.device(), ", tokens on ", dev);
  p.pages = k.size(0);
  p.heads = k.size(1);
  p.page = k.size(2);
  p.d = k.size(3);
  if (p.kind == VQ2_I8) {
    for (const at::Tensor* s : {ks, vs})
      if (!s || s->scalar_type() != at::kFloat || s->dim() != 3 || s->size(0) != p.pages || s->size(1) != p.heads ||
          s->size(2) != p.page || !s->is_contiguous() || s->device() != dev)
        refuse("int8 pools need contiguous fp32 k_scale and v_scale [pages, kv_heads, page_size]");
    p.ks = static_cast<float*>(ks->data_ptr());
    p.vs = static_cast<float*>(vs->data_ptr());
  } else if (ks || vs) {
    refuse("scales go with int8 pools only");
  } else if (dtype >= 0 && p.kind != dtype) {
    refuse("pools hold ", k.scalar_type(), ", which is not the tokens' type");
  }
  if ((heads >= 0 && p.heads != heads) || (d >= 0 && p.d != d))
    refuse("pools have ", p.heads, " heads of ", p.d, "; the tokens ", heads < 0 ? p.heads : heads, " of ", d < 0 ? p.d : d);
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.device() != dev || (table.size(1) > 1 && table.stride(1) != 1))
    refuse("table must be int32 [seqs, cols] with contiguous rows, on the tokens' device");
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.table = static_cast<const int32_t*>(table.const_data_ptr());
  p.seqs = table.size(0);
  p.cols = table.size(1);
  p.stride = table.stride(0);   // 0 where sequences share one row
  return p;
}

const float* frequencies(const at::Tensor& f, int64_t d, c10::Device dev, int64_t& rot) {
  if (f.scalar_type() != at::kFloat || f.dim() != 1 || !f.is_contiguous() || f.device() != dev)
    refuse("inv_freq must be a contiguous fp32 vector on the tokens' device");
  rot = 2 * f.size(0);
  if (rot < 2 || rot > d) refuse("inv_freq turns ", rot, " values of a head of ", d);
  return static_cast<const float*>(f.const_data_ptr());
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType t, c10::Device dev) {
  return at::detail::empty_cuda(sizes, at::TensorOptions().dtype(t).device(dev));
}

void* current_stream(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void check(int status, const char* name) {
  if (status == VQ2_OK) return;
  PyObject* r = PyObject_CallFunction(check_status, "is", status, name);
  if (!r) throw Raised();
  Py_DECREF(r);
  throw std::runtime_error(name);
}

PyObject* pair(PyObject* a, PyObject* b) {   // steals both
  PyObject* t = PyTuple_New(2);
  if (!t) {
    Py_DECREF(a);
    Py_DECREF(b);
    throw Raised();
  }
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}
PyObject* none() {
  Py_INCREF(Py_None);
  return Py_None;
}

// q, k|None, positions, inv_freq, interleaved, factor, inverse -> (q', k'|None)
PyObject* rotary(PyObject* const* a) {
  const at::Tensor q = rows(tensor(a[0], "q"), "q");
  const at::Tensor* k0 = maybe(a[1], "k");
  const at::Tensor &pos0 = tensor(a[2], "positions"), &f = tensor(a[3], "inv_freq");
  const auto dev = q.device();
  const int64_t T = q.size(0), d = q.size(2);
  if (pos0.dim() != 1 || pos0.size(0) != T || (pos0.scalar_type() != at::kInt && pos0.scalar_type() != at::kLong) || pos0.device() != dev)
    refuse("positions must be int32 or int64 [", T, "] on ", dev, "; got ", pos0.scalar_type(), " ", pos0.sizes());
  int64_t rot;
  const float* fp = frequencies(f, d, dev, rot);
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor pos = pos0.contiguous();
  at::Tensor q_out = empty({T, q.size(1), d}, q.scalar_type(), dev), k, k_out;
  if (k0) {
    k = rows(*k0, "k", &q);
    k_out = empty({T, k.size(1), d}, q.scalar_type(), dev);
  }
  if (T)
    check(f_rotary(q.const_data_ptr(), q.stride(0), q.stride(1), q.size(1), k0 ? k.const_data_ptr() : nullptr,
                   k0 ? k.stride(0) : 0, k0 ? k.stride(1) : 0, k0 ? k.size(1) : 0, code(q.scalar_type()), T, d,
                   pos.const_data_ptr(), pos.scalar_type() == at::kLong, fp, rot, truth(a[4]), (float)number(a[5]),
                   truth(a[6]), q_out.data_ptr(), k0 ? k_out.data_ptr() : nullptr, current_stream(dev)),
          "vq2_rotary");
  return pair(THPVariable_Wrap(std::move(q_out)), k0 ? THPVariable_Wrap(std::move(k_out)) : none());
}

// k, v, (k_pages, v_pages, table, k_scale, v_scale), lens, starts, q, inv_freq, interleaved, factor -> q'|None
PyObject* cache_write(PyObject* const* a) {
  const at::Tensor k = rows(tensor(a[0], "k"), "k"), v = rows(tensor(a[1], "v"), "v", &k);
  const auto dev = k.device();
  const int64_t T = k.size(0), d = k.size(2);
  const int dtype = code(k.scalar_type());
  const Pools p = pools(a + 2, dtype, k.size(1), d, dev);
  if (v.size(1) != k.size(1)) refuse("k and v must have the same heads");
  const int32_t* lens = ints(tensor(a[7], "lens"), "lens", p.seqs, dev);
  const at::Tensor* starts = maybe(a[8], "starts");
  if (!starts && T != p.seqs)
    refuse("without starts every sequence has one new token; got ", T, " tokens for ", p.seqs, " sequences");
  const int32_t* starts_p = starts ? ints(*starts, "starts", p.seqs + 1, dev) : nullptr;
  const at::Tensor *f = maybe(a[10], "inv_freq"), *q0 = maybe(a[9], "q");
  int64_t rot = 0;
  const float* fp = f ? frequencies(*f, d, dev, rot) : nullptr;
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor q, q_out;
  if (q0) {
    q = rows(*q0, "q", &k);
    q_out = empty({T, q.size(1), d}, q.scalar_type(), dev);
  }
  if (T)
    check(f_write(q0 ? q.const_data_ptr() : nullptr, q0 ? q.stride(0) : 0, q0 ? q.stride(1) : 0, q0 ? q.size(1) : 0,
                  q0 ? q_out.data_ptr() : nullptr, k.const_data_ptr(), k.stride(0), k.stride(1), v.const_data_ptr(),
                  v.stride(0), v.stride(1), dtype, T, fp, rot, truth(a[11]), (float)number(a[12]), p.k, p.v, p.kind, p.ks,
                  p.vs, p.pages, p.heads, p.page, p.d, p.table, p.stride, p.cols, lens, starts_p, p.seqs,
                  current_stream(dev)),
          "vq2_cache_write");
  return q0 ? THPVariable_Wrap(std::move(q_out)) : none();
}

// (k_pages, v_pages, table, k_scale, v_scale), starts, total, dtype|None -> (k, v)
PyObject* cache_read(PyObject* const* a) {
  const at::Tensor& k_pages = tensor(a[0], "k_pages");
  on_cuda(k_pages);
  const auto dev = k_pages.device();
  at::ScalarType t = k_pages.scalar_type() == at::kChar ? at::kBFloat16 : k_pages.scalar_type();
  if (a[7] != Py_None) {
    if (!THPDtype_Check(a[7])) refuse("dtype must be a torch dtype");
    t = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
  }
  if (t != at::kHalf && t != at::kBFloat16) refuse("a cache is read back as fp16 or bf16; got ", t);
  const Pools p = pools(a, code(t), -1, -1, dev);
  const int32_t* starts = ints(tensor(a[5], "starts"), "starts", p.seqs + 1, dev);
  const int64_t total = integer(a[6]);
  if (total < 0) refuse("total counts tokens: it is not negative");
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor k = empty({total, p.heads, p.d}, t, dev), v = empty({total, p.heads, p.d}, t, dev);
  if (total)
    check(f_read(p.k, p.v, p.kind, p.ks, p.vs, p.pages, p.heads, p.page, p.d, p.table, p.stride, p.cols, starts, p.seqs,
                 k.data_ptr(), v.data_ptr(), code(t), total, current_stream(dev)),
          "vq2_cache_read");
  return pair(THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
}

// q, (k_pages, v_pages, table, k_scale, v_scale), lens, starts, scale|None, causal, window, max_new|None,
// max_len|None, return_lse -> out | (out, lse)
PyObject* paged_attention(PyObject* const* a) {
  at::Tensor q = rows(tensor(a[0], "q"), "q");
  const auto dev = q.device();
  const int64_t T = q.size(0), hq = q.size(1), d = q.size(2);
  const int dtype = code(q.scalar_type());
  const Pools p = pools(a + 1, dtype, -1, d, dev);
  if (!hq || !p.heads || hq % p.heads) refuse(hq, " query heads do not share ", p.heads, " key/value heads");
  const int32_t* lens = ints(tensor(a[6], "lens"), "lens", p.seqs, dev);
  const at::Tensor* starts = maybe(a[7], "starts");
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)d) : number(a[8]);
  const int causal = truth(a[9]), want_lse = truth(a[13]);
  const int64_t window = integer(a[10]), room = p.cols * p.page;
  int64_t max_new = a[11] == Py_None ? T : std::min(integer(a[11]), T);
  const int64_t max_len = a[12] == Py_None ? room : std::min(integer(a[12]), room);
  const int32_t* starts_p = nullptr;
  if (!starts) {
    if (T != p.seqs)
      refuse("without starts every sequence has one new token; got ", T, " tokens for ", p.seqs, " sequences");
    max_new = 1;
  } else {
    starts_p = ints(*starts, "starts", p.seqs + 1, dev);
  }
  if (window < 0 || max_new < 0 || max_len < 0) refuse("window, max_new and max_len count tokens: none is negative");
  const c10::cuda::CUDAGuard guard(dev);
  if (reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 || q.stride(0) % 8 || q.stride(1) % 8)
    q = q.clone(at::MemoryFormat::Contiguous);   // the kernels read 16 bytes at a time
  at::Tensor out = empty({T, hq, d}, q.scalar_type(), dev), lse, ws;
  if (want_lse) lse = empty({T, hq}, at::kFloat, dev);
  if (T) {
    const int64_t bytes = f_workspace(T, hq, p.heads, d, p.kind, p.seqs, max_new, max_len, window);
    if (bytes) ws = empty({bytes}, at::kByte, dev);
    check(f_attention(q.const_data_ptr(), q.stride(0), q.stride(1), dtype, T, hq, p.k, p.v, p.kind, p.ks, p.vs, p.pages,
                      p.heads, p.page, p.d, p.table, p.stride, p.cols, lens, starts_p, p.seqs, max_new, max_len, (float)scale,
                      causal, window, out.data_ptr(), want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr,
                      bytes ? ws.data_ptr() : nullptr, bytes, current_stream(dev)),
          "vq2_paged_attention");
  }
  if (!want_lse) return THPVariable_Wrap(std::move(out));
  return pair(THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
}

// No C++ exception leaves an entry of the module.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != N) refuse("expected ", N, " arguments, got ", n);
    return F(args);
  } catch (const Raised&) {
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

// bind({name: address}, check, OutOfMemoryError)
PyObject* bind(PyObject*, PyObject* args) {
  PyObject *addresses, *checker, *oom;
  if (!PyArg_ParseTuple(args, "O!OO", &PyDict_Type, &addresses, &checker, &oom)) return nullptr;
  auto of = [&](const char* name) -> void* {
    PyObject* v = PyDict_GetItemString(addresses, name);
    return v ? PyLong_AsVoidPtr(v) : nullptr;
  };
  f_rotary = reinterpret_cast<decltype(f_rotary)>(of("vq2_rotary"));
  f_write = reinterpret_cast<decltype(f_write)>(of("vq2_cache_write"));
  f_read = reinterpret_cast<decltype(f_read)>(of("vq2_cache_read"));
  f_attention = reinterpret_cast<decltype(f_attention)>(of("vq2_paged_attention"));
  f_workspace = reinterpret_cast<decltype(f_workspace)>(of("vq2_paged_attention_workspace"));
  if (!f_rotary || !f_write || !f_read || !f_attention || !f_workspace) {
    PyErr_SetString(PyExc_ValueError, "an entry point's address is missing");
    return nullptr;
  }
  Py_INCREF(checker);
  Py_XSETREF(check_status, checker);
  Py_INCREF(oom);
  Py_XSETREF(out_of_memory, oom);
  return none();
}

#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(rotary, 7), ENTRY(cache_write, 13), ENTRY(cache_read, 8), ENTRY(paged_attention, 14),
                         {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention_host() { return PyModule_Create(&module); }
