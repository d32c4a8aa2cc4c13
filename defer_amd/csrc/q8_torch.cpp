// q8_torch.cpp -- the 8-bit operators on torch tensors (defer_amd.q8): checks,
// outputs, the call on torch's current stream. A call for one token is a few
// microseconds on the GPU, so what Python would take for the same checks (4 to 7
// us a call) is most of it.
//
// Nothing is kept between calls but the library's functions. Every refusal is
// a ValueError raised before anything is allocated or queued; what the
// library refuses goes to Python's own error of that library.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <dlfcn.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/defer_gpu.h"
#include "q8_index.h"

namespace {

using at::IntArrayRef;
using at::ScalarType;
using at::Tensor;

constexpr int64_t PAGE = 64;

struct {
  decltype(&defer_gpu_q8_quantize) quantize;
  decltype(&defer_gpu_q8_rms_norm) rms_norm;
  decltype(&defer_gpu_q8_linear) linear;
  decltype(&defer_gpu_q8_kv_write) kv_write;
  decltype(&defer_gpu_q8_kv_read) kv_read;
  decltype(&defer_gpu_q8_attention_workspace) attention_workspace;
  decltype(&defer_gpu_q8_attention) attention;
  PyObject* stream_of;  // device -> raw current stream
  PyObject* check;      // raises for a code that is not OK
  PyObject* out_of_memory;
} lib;

struct Refused : std::invalid_argument {
  using std::invalid_argument::invalid_argument;
};
struct PythonError {};  // already set

void need(bool ok, const std::string& why) {
  if (!ok) throw Refused(why);
}

std::string shape_of(IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Refused(std::string(what) + " is not a tensor but " + Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  if (c10::GradMode::is_enabled() && t.requires_grad())  // its gradient would be lost without a word
    throw Refused(std::string(what) + " requires a gradient, and there is no backward: detach it or call under torch.no_grad()");
  return t;
}

// The call has written this tensor: autograd sees that what it may have saved is gone.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const Tensor& on_gpu(PyObject* o, const char* what) {
  const Tensor& t = tensor(o, what);
  if (!t.is_cuda()) throw Refused(std::string(what) + " is not a tensor on a GPU");
  return t;
}

void expect(const Tensor& t, const char* what, at::Device dev, ScalarType type, IntArrayRef shape) {
  if (t.layout() == at::kStrided && t.device() == dev && t.scalar_type() == type && t.sizes() == shape) return;
  throw Refused(std::string(what) + ": need a " + c10::toString(type) + " tensor of shape " + shape_of(shape) + " on " +
                dev.str() + ", got " + c10::toString(t.scalar_type()) + " " + shape_of(t.sizes()) + " on " + t.device().str());
}

// The address of a contiguous tensor of this device, type and shape.
template <class T>
T* take(PyObject* o, const char* what, at::Device dev, ScalarType type, IntArrayRef shape) {
  const Tensor& t = tensor(o, what);
  expect(t, what, dev, type, shape);
  if (!t.is_contiguous()) throw Refused(std::string(what) + " is not contiguous");
  return static_cast<T*>(t.data_ptr());
}

// Rows of contiguous values any distance apart: that distance.
int64_t row_stride(const Tensor& t, const char* what, at::Device dev, ScalarType type, IntArrayRef shape) {
  expect(t, what, dev, type, shape);
  int64_t n = 1;
  bool dense = true;
  for (size_t i = shape.size() - 1; i >= 1; --i) {
    dense = dense && (shape[i] == 1 || t.stride(i) == n);
    n *= shape[i];
  }
  if (t.is_contiguous()) return n;
  if (!dense) throw Refused(std::string(what) + ": the values of a row are not contiguous");
  if (shape[0] <= 1) return n;
  if (t.stride(0) < n) throw Refused(std::string(what) + ": rows overlap");
  return t.stride(0);
}

// Rows that a call writes lie apart from those it reads, or are the same rows.
void apart(const Tensor& out, int64_t os, const Tensor& in, int64_t is, const char* what) {
  const int64_t rows = out.size(0), v = out.element_size(), n = rows ? out.numel() / rows * v : 0;
  if (rows <= 0xffffffffll && q8::overlap(out.data_ptr(), os * v, (uint32_t)rows, in.data_ptr(), is * v, (uint32_t)rows, n))
    throw Refused(std::string("out overlaps ") + what);
}

uint32_t u32(int64_t n, const char* what) {
  if (n < 0 || n > 0xffffffffll) throw Refused(std::string(what) + " is out of range: " + std::to_string(n));
  return (uint32_t)n;
}

uint32_t value_type(ScalarType t, const char* what) {
  if (t == ScalarType::Float) return DEFER_GPU_F32;
  if (t == ScalarType::BFloat16) return DEFER_GPU_BF16;
  if (t == ScalarType::Half) return DEFER_GPU_F16;
  throw Refused(std::string(what) + ": float32, bfloat16 or float16, not " + c10::toString(t));
}
ScalarType dtype(PyObject* o) {
  if (!THPDtype_Check(o)) throw Refused(std::string("dtype: not a torch.dtype but ") + Py_TYPE(o)->tp_name);
  const ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  (void)value_type(t, "dtype");
  return t;
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError();
  return (float)v;
}

Tensor fresh(IntArrayRef shape, ScalarType type, at::Device dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
}

// f(stream) with the tensors' device current and torch's current stream there.
template <class F>
void call(at::Device dev, F f) {
  const c10::DeviceGuard guard(dev);
  PyObject* const index = PyLong_FromLong(dev.index());
  if (!index) throw PythonError();
  PyObject* const s = PyObject_CallOneArg(lib.stream_of, index);
  Py_DECREF(index);
  if (!s) throw PythonError();
  void* const stream = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if (PyErr_Occurred()) throw PythonError();
  int rc;
  Py_BEGIN_ALLOW_THREADS;  // a launch waits where the queue is full
  rc = f(stream);
  Py_END_ALLOW_THREADS;
  if (rc == DEFER_GPU_OK) return;
  PyObject* const code = PyLong_FromLong(rc);
  PyObject* const r = code ? PyObject_CallOneArg(lib.check, code) : nullptr;
  Py_XDECREF(code);
  if (r) {  // it always raises
    Py_DECREF(r);
    throw Refused("error " + std::to_string(rc));
  }
  throw PythonError();
}

PyObject* tuple(const Tensor& a, const Tensor& b) {
  return Py_BuildValue("(NN)", THPVariable_Wrap(a), THPVariable_Wrap(b));
}

// The pool and the table (a tuple of five), and the call's rows.
struct Cache {
  defer_gpu_q8_pages p;
  defer_gpu_q8_rows r;

  Cache(PyObject* pages, int64_t head_dim, at::Device dev) {
    need(PyTuple_Check(pages) && PyTuple_GET_SIZE(pages) == 5, "pages: need Pages");
    PyObject** const o = &PyTuple_GET_ITEM(pages, 0);
    const Tensor &keys = tensor(o[0], "keys"), &table = tensor(o[4], "table");
    need(keys.dim() == 4, "keys: need [pages, heads, 64, D]");
    need(table.dim() == 2, "table: need [sequences, width]");
    const int64_t n = keys.size(0), heads = keys.size(1), d = keys.size(3);
    if (!(head_dim >= 1 && head_dim <= d && d == (head_dim + PAGE - 1) / PAGE * PAGE))
      throw Refused("head size " + std::to_string(head_dim) + " in pages of " + std::to_string(d));
    p.keys = take<int8_t>(o[0], "keys", dev, ScalarType::Char, {n, heads, PAGE, d});
    p.values = take<int8_t>(o[1], "values", dev, ScalarType::Char, {n, heads, d, PAGE});
    p.key_scale = take<float>(o[2], "key_scale", dev, ScalarType::Float, {n, heads, PAGE});
    p.value_scale = take<float>(o[3], "value_scale", dev, ScalarType::Float, {n, heads, PAGE});
    p.table = take<int32_t>(o[4], "table", dev, ScalarType::Int, table.sizes());
    p.pages = u32(n, "pages");
    p.heads = u32(heads, "heads");
    p.head_dim = (uint32_t)head_dim;
    p.table_width = u32(table.size(1), "table");
    r.sequences = u32(table.size(0), "sequences");
  }
  void rows(PyObject* kv_len, PyObject* row_start, int64_t n, PyObject* most_rows, at::Device dev) {
    const int64_t most = most_rows != Py_None ? integer(most_rows) : row_start != Py_None ? n : std::min<int64_t>(n, 1);
    if (!(most >= 0 && most <= n)) throw Refused("most_rows " + std::to_string(most) + " of " + std::to_string(n) + " rows");
    r.row_start = nullptr;
    if (row_start != Py_None)
      r.row_start = take<int32_t>(row_start, "row_start", dev, ScalarType::Int, {(int64_t)r.sequences + 1});
    else if (n != (int64_t)r.sequences)
      throw Refused(std::to_string(n) + " rows of " + std::to_string(r.sequences) + " sequences without row_start");
    r.kv_len = take<int32_t>(kv_len, "kv_len", dev, ScalarType::Int, {(int64_t)r.sequences});
    r.rows = u32(n, "rows");
    r.most_rows = (uint32_t)most;
  }
};

// ------------------------------------------------------------- operators

PyObject* quantize(PyObject* const* a) {
  const Tensor& x = on_gpu(a[0], "x");
  const uint32_t ty = value_type(x.scalar_type(), "x");
  need(x.dim() == 2 && x.size(1) > 0, "x: need [rows, n]");
  const auto dev = x.device();
  const int64_t st = row_stride(x, "x", dev, x.scalar_type(), x.sizes());
  const uint32_t rows = u32(x.size(0), "rows"), n = u32(x.size(1), "n");
  const Tensor codes = fresh(x.sizes(), ScalarType::Char, dev), scale = fresh({x.size(0)}, ScalarType::Float, dev);
  call(dev, [&](void* s) {
    return lib.quantize(ty, x.data_ptr(), st, rows, n, codes.data_ptr<int8_t>(), scale.data_ptr<float>(), s);
  });
  return tuple(codes, scale);
}

PyObject* rms_norm(PyObject* const* a) {  // x, weight, eps, residual, out
  const Tensor& x = on_gpu(a[0], "x");
  const ScalarType type = x.scalar_type();
  const uint32_t ty = value_type(type, "x");
  need(x.dim() == 2 && x.size(1) > 0, "x: need [rows, n]");
  const auto dev = x.device();
  const uint32_t rows = u32(x.size(0), "rows"), n = u32(x.size(1), "n");
  const int64_t xs = row_stride(x, "x", dev, type, x.sizes());
  const void* const w = take<void>(a[1], "weight", dev, type, {x.size(1)});
  const float eps = real(a[2]);
  const void* r = nullptr;
  int64_t rs = 0, zs = 0;
  Tensor z = x;
  bool store = false;
  if (a[3] != Py_None) {
    const Tensor& t = tensor(a[3], "residual");
    rs = row_stride(t, "residual", dev, type, x.sizes());
    r = t.data_ptr();
  }
  if (a[4] != Py_None) {
    z = tensor(a[4], "out");
    zs = row_stride(z, "out", dev, type, x.sizes());
    store = true;
    apart(z, zs, x, xs, "x");
    if (r) apart(z, zs, tensor(a[3], "residual"), rs, "residual");
  } else if (a[3] != Py_None) {
    z = fresh(x.sizes(), type, dev);
    zs = n;
    store = true;
  }
  const Tensor codes = fresh(x.sizes(), ScalarType::Char, dev), scale = fresh({x.size(0)}, ScalarType::Float, dev);
  call(dev, [&](void* s) {
    return lib.rms_norm(ty, x.data_ptr(), xs, r, rs, w, eps, rows, n, store ? z.data_ptr() : nullptr, zs,
                        codes.data_ptr<int8_t>(), scale.data_ptr<float>(), s);
  });
  if (store) written(z);
  PyObject* const zo = a[4] != Py_None ? a[4] : store ? nullptr : a[0];  // the caller's own tensor comes back as it is
  Py_XINCREF(zo);
  return Py_BuildValue("(NNN)", zo ? zo : THPVariable_Wrap(z), THPVariable_Wrap(codes), THPVariable_Wrap(scale));
}

PyObject* linear(PyObject* const* a) {  // x, x_scale, w, w_scale, dtype
  const Tensor& x = on_gpu(a[0], "x");
  const Tensor& w = tensor(a[2], "w");
  const ScalarType type = dtype(a[4]);
  need(x.dim() == 2 && w.dim() == 2, "need x [rows, k] and w [m, k]");
  const auto dev = x.device();
  const int64_t rows = x.size(0), k = x.size(1), m = w.size(0);
  const int64_t xst = row_stride(x, "x", dev, ScalarType::Char, x.sizes());
  const int64_t wst = row_stride(w, "w", dev, ScalarType::Char, {m, k});
  const float* const xs = take<float>(a[1], "x_scale", dev, ScalarType::Float, {rows});
  const float* const ws = take<float>(a[3], "w_scale", dev, ScalarType::Float, {m});
  const uint32_t r32 = u32(rows, "rows"), m32 = u32(m, "m"), k32 = u32(k, "k");
  const Tensor y = fresh({rows, m}, type, dev);
  call(dev, [&](void* s) {
    return lib.linear(x.data_ptr<int8_t>(), xst, xs, w.data_ptr<int8_t>(), wst, ws, r32, m32, k32, value_type(type, "dtype"),
                      y.data_ptr(), m, s);
  });
  return THPVariable_Wrap(y);
}

PyObject* kv_write(PyObject* const* a) {  // pages, k, v, kv_len, row_start, most_rows
  const Tensor& k = on_gpu(a[1], "k");
  const Tensor& v = tensor(a[2], "v");
  const uint32_t ty = value_type(k.scalar_type(), "k");
  need(k.dim() == 3, "k: need [rows, heads, head_dim]");
  const auto dev = k.device();
  Cache c(a[0], k.size(2), dev);
  if (k.size(1) != (int64_t)c.p.heads)
    throw Refused("k has " + std::to_string(k.size(1)) + " heads, the pages " + std::to_string(c.p.heads));
  const int64_t ks = row_stride(k, "k", dev, k.scalar_type(), k.sizes());
  const int64_t vs = row_stride(v, "v", dev, k.scalar_type(), k.sizes());
  c.rows(a[3], a[4], k.size(0), a[5], dev);
  call(dev, [&](void* s) { return lib.kv_write(&c.p, &c.r, ty, k.data_ptr(), ks, v.data_ptr(), vs, s); });
  for (Py_ssize_t i = 0; i < 4; ++i) written(THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i)));
  Py_RETURN_NONE;
}

PyObject* kv_read(PyObject* const* a) {  // pages, kv_len, row_start, rows, head_dim, most_rows, dtype
  const auto dev = on_gpu(a[1], "kv_len").device();
  const ScalarType type = dtype(a[6]);
  const int64_t rows = integer(a[3]), hd = integer(a[4]);
  Cache c(a[0], hd, dev);
  c.rows(a[1], a[2], rows, a[5], dev);
  const Tensor k = fresh({rows, c.p.heads, hd}, type, dev), v = fresh({rows, c.p.heads, hd}, type, dev);
  call(dev, [&](void* s) { return lib.kv_read(&c.p, &c.r, value_type(type, "dtype"), k.data_ptr(), v.data_ptr(), s); });
  return tuple(k, v);
}

PyObject* attention(PyObject* const* a) {  // q, pages, kv_len, row_start, most_rows, most_len, scale, hidden, out
  const Tensor& q = on_gpu(a[0], "q");
  const ScalarType type = q.scalar_type();
  const uint32_t ty = value_type(type, "q");
  need(q.dim() == 3, "q: need [rows, heads, head_dim]");
  const auto dev = q.device();
  const int64_t rows = q.size(0), hd = q.size(2), n = q.size(1) * hd;
  const uint32_t heads = u32(q.size(1), "heads");
  Cache c(a[1], hd, dev);
  const int64_t qs = row_stride(q, "q", dev, type, q.sizes());
  c.rows(a[2], a[3], rows, a[4], dev);
  const int64_t most_len = a[5] != Py_None ? integer(a[5]) : std::min<int64_t>(PAGE * c.p.table_width, 0x7fffffff);
  if (!(most_len >= 0 && most_len <= 0x7fffffff)) throw Refused("most_len " + std::to_string(most_len));
  const float scale = a[6] != Py_None ? real(a[6]) : (float)std::pow((double)hd, -0.5);
  const uint8_t* hidden = nullptr;
  int64_t hs = 0;
  uint32_t hn = 0;
  if (a[7] != Py_None) {
    const Tensor& h = tensor(a[7], "hidden");
    need((h.scalar_type() == ScalarType::Byte || h.scalar_type() == ScalarType::Bool) && h.dim() == 2,
         "hidden: need [sequences, n] uint8 or bool");
    hn = u32(h.size(1), "hidden");
    hs = row_stride(h, "hidden", dev, h.scalar_type(), {(int64_t)c.r.sequences, h.size(1)});
    hidden = static_cast<const uint8_t*>(h.data_ptr());
  }
  const bool clear = a[8] == Py_None;
  Tensor out;
  int64_t os = n;
  if (clear) {
    out = fresh(q.sizes(), type, dev);
  } else {
    out = tensor(a[8], "out");
    os = row_stride(out, "out", dev, type, q.sizes());
    apart(out, os, q, qs, "q");
  }
  const size_t need_bytes = lib.attention_workspace(&c.p, &c.r, heads, (uint32_t)most_len);
  Tensor work;
  if (need_bytes) work = fresh({(int64_t)need_bytes}, ScalarType::Byte, dev);
  call(dev, [&](void* s) {
    return lib.attention(&c.p, &c.r, ty, q.data_ptr(), qs, heads, (uint32_t)most_len, scale, hidden, hs, hn, out.data_ptr(),
                         os, clear, need_bytes ? work.data_ptr() : nullptr, need_bytes, s);
  });
  if (clear) return THPVariable_Wrap(out);
  written(out);
  Py_INCREF(a[8]);
  return a[8];
}

// A call from Python: the argument count, and no C++ exception gets out.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) return PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
  if (!lib.attention) return PyErr_Format(PyExc_RuntimeError, "bind() first");
  try {
    need(!at::tracer::impl::is_dispatch_enabled(), "torch.jit.trace would keep what this call returns as constants");
    return F(args);
  } catch (const PythonError&) {
    return nullptr;
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(lib.out_of_memory, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// bind(path of the loaded library, stream_of, check, out_of_memory)
PyObject* bind(PyObject*, PyObject* args) {
  const char* path;
  PyObject *stream_of, *check, *out_of_memory;
  if (!PyArg_ParseTuple(args, "sOOO", &path, &stream_of, &check, &out_of_memory)) return nullptr;
  void* const h = dlopen(path, RTLD_NOW | RTLD_NOLOAD);
  if (!h) return PyErr_Format(PyExc_ImportError, "%s is not loaded", path);
  auto take = [&](const char* name, auto& f) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(h, name));
    if (!f) PyErr_Format(PyExc_ImportError, "%s has no %s", path, name);
    return f != nullptr;
  };
  if (!(take("defer_gpu_q8_quantize", lib.quantize) && take("defer_gpu_q8_rms_norm", lib.rms_norm) &&
        take("defer_gpu_q8_linear", lib.linear) && take("defer_gpu_q8_kv_write", lib.kv_write) &&
        take("defer_gpu_q8_kv_read", lib.kv_read) &&
        take("defer_gpu_q8_attention_workspace", lib.attention_workspace)))
    return nullptr;
  Py_INCREF(stream_of);
  Py_INCREF(check);
  Py_INCREF(out_of_memory);
  lib.stream_of = stream_of;
  lib.check = check;
  lib.out_of_memory = out_of_memory;
  if (!take("defer_gpu_q8_attention", lib.attention)) return nullptr;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<quantize, 1>("quantize"), method<rms_norm, 5>("rms_norm"), method<linear, 5>("linear"),
                         method<kv_write, 6>("kv_write"), method<kv_read, 7>("kv_read"),
                         method<attention, 9>("attention"), {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_q8_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__q8_torch() { return PyModule_Create(&module); }
