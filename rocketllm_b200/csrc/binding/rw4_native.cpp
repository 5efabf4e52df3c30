// Host fast path of the 8-bit operators' Python entry points (rocketllm_b200/kernels.py).
//
// A decode-sized call of these operators takes 1.5 to 8 us on the GPU; checking its arguments,
// allocating its results and marshalling a dozen values through ctypes takes 9 to 19 us in Python
// and 3.5 to 5 us here (of which the launch itself is 2.1).  Each function takes the plain case --
// CUDA tensors of the documented types and shapes, all on the current device, results to be
// allocated -- makes the same C-ABI call (include/rw4.h) on the current stream and returns the
// results.  For anything else it returns None and has launched nothing: the Python entry point then
// goes on with its own checks, which make the errors, the compact copies, the writes into given
// outputs and the calls on other devices.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "rw4.h"

namespace {

constexpr int64_t kMaxRow = 131056;

// A strided CUDA tensor on device `dev` (any device when dev < 0), not a deferred kind.
bool plain(PyObject* o, int dev) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg() &&
         (dev < 0 || t.get_device() == dev);
}

int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return RW4_F32;
  if (t == at::kBFloat16) return RW4_BF16;
  if (t == at::kHalf) return RW4_F16;
  return -1;
}

// t [..., K] as rows with one stride between them, without a copy (the halves of a [B, S, 2 K]
// projection are such rows).
bool as_rows(const at::Tensor& t, int64_t& m, int64_t& k, int64_t& ld) {
  const int64_t d = t.dim();
  if (d < 1) return false;
  k = t.size(d - 1);
  if (k < 1 || k > kMaxRow || t.stride(d - 1) != 1) return false;
  if (d == 2) {
    m = t.size(0);
    ld = t.stride(0);
    return true;
  }
  m = 1;
  ld = k;
  for (int64_t i = d - 2; i >= 0; --i) {   // outwards; m rows so far, ld apart
    const int64_t n = t.size(i);
    if (n != 1 && m == 1) ld = t.stride(i);
    else if (n > 1 && m > 1 && t.stride(i) != m * ld) return false;
    m *= n;
  }
  return true;
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, c10::Device dev) {
  return at::detail::empty_cuda(sizes, dtype, dev, std::nullopt);
}

struct Call {
  int dev;
  void* stream;
};

// The current device is `dev`; its current stream.
bool here(int dev, Call& c) {
  c.dev = dev;
  if (c10::cuda::current_device() != dev) return false;
  c.stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  return true;
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// int8_quantize(x, gate or None)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !plain(a[0], -1)) return none();
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const int dev = x.get_device(), code = dtype_code(x.scalar_type());
  int64_t m, k, ld, gm, gk, gld = 0;
  Call c;
  if (code < 0 || !as_rows(x, m, k, ld) || !here(dev, c)) return none();
  const void* gate = nullptr;
  if (a[1] != Py_None) {
    if (!plain(a[1], dev)) return none();
    const at::Tensor& g = THPVariable_Unpack(a[1]);
    if (g.scalar_type() != x.scalar_type() || g.sizes() != x.sizes() || !as_rows(g, gm, gk, gld))
      return none();
    gate = g.const_data_ptr();
  }
  at::Tensor codes = empty(x.sizes(), at::kChar, x.device());
  at::Tensor scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x.device());
  int st;
  const void* xp = x.const_data_ptr();
  int8_t* cp = static_cast<int8_t*>(codes.mutable_data_ptr());
  float* sp = static_cast<float*>(scale.mutable_data_ptr());
  Py_BEGIN_ALLOW_THREADS
  st = rw4_int8_quantize(xp, ld, gate, gld, code, m, k, cp, sp, c.stream);
  Py_END_ALLOW_THREADS
  return st == RW4_OK ? tuple_of({codes, scale}) : none();
  END_HANDLE_TH_ERRORS
}

// int8_rmsnorm(x, weight, eps, residual or None)
PyObject* rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !plain(a[0], -1) || !PyFloat_Check(a[2])) return none();
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const int dev = x.get_device(), code = dtype_code(x.scalar_type());
  int64_t m, k, ld, rm, rk, rld = 0;
  Call c;
  if (code < 0 || !as_rows(x, m, k, ld) || !plain(a[1], dev) || !here(dev, c)) return none();
  const at::Tensor& w = THPVariable_Unpack(a[1]);
  if (w.scalar_type() != x.scalar_type() || w.dim() != 1 || w.size(0) != k || !w.is_contiguous())
    return none();
  const void* residual = nullptr;
  if (a[3] != Py_None) {
    if (!plain(a[3], dev)) return none();
    const at::Tensor& r = THPVariable_Unpack(a[3]);
    if (r.scalar_type() != x.scalar_type() || r.sizes() != x.sizes() || !as_rows(r, rm, rk, rld))
      return none();
    residual = r.const_data_ptr();
  }
  at::Tensor hidden;
  if (residual || a[3] != Py_None) hidden = empty(x.sizes(), x.scalar_type(), x.device());
  at::Tensor codes = empty(x.sizes(), at::kChar, x.device());
  at::Tensor scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x.device());
  const float eps = static_cast<float>(PyFloat_AS_DOUBLE(a[2]));
  int st;
  const void *xp = x.const_data_ptr(), *wp = w.const_data_ptr();
  void* hp = hidden.defined() ? hidden.mutable_data_ptr() : nullptr;
  int8_t* cp = static_cast<int8_t*>(codes.mutable_data_ptr());
  float* sp = static_cast<float*>(scale.mutable_data_ptr());
  Py_BEGIN_ALLOW_THREADS
  st = rw4_int8_rmsnorm(xp, ld, residual, rld, wp, code, m, k, eps, hp, cp, sp, c.stream);
  Py_END_ALLOW_THREADS
  if (st != RW4_OK) return none();
  return hidden.defined() ? tuple_of({codes, scale, hidden}) : tuple_of({codes, scale});
  END_HANDLE_TH_ERRORS
}

// int8 codes [..., K] and their float32 scale, one a row, both contiguous on `dev`.
bool codes_ok(const at::Tensor& c, PyObject* scale, int dev, int64_t& m) {
  if (!plain(scale, dev)) return false;
  const at::Tensor& s = THPVariable_Unpack(scale);
  if (c.scalar_type() != at::kChar || s.scalar_type() != at::kFloat || c.dim() < 1 ||
      !c.is_contiguous() || !s.is_contiguous())
    return false;
  const auto rows = c.sizes().slice(0, c.dim() - 1);
  const auto ss = s.sizes();
  const bool column = ss.size() == rows.size() + 1 && ss.back() == 1;
  if (ss != rows && !(column && ss.slice(0, rows.size()) == rows)) return false;
  m = s.numel();
  return true;
}

// int8_dequantize(codes, scale, dtype)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !plain(a[0], -1) || !THPDtype_Check(a[2])) return none();
  const at::Tensor& codes = THPVariable_Unpack(a[0]);
  const at::ScalarType dt = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
  const int dev = codes.get_device(), code = dtype_code(dt);
  int64_t m;
  Call c;
  if (code < 0 || !codes_ok(codes, a[1], dev, m) || !here(dev, c)) return none();
  at::Tensor out = empty(codes.sizes(), dt, codes.device());
  int st;
  const int8_t* cp = static_cast<const int8_t*>(codes.const_data_ptr());
  const float* sp = static_cast<const float*>(THPVariable_Unpack(a[1]).const_data_ptr());
  void* op = out.mutable_data_ptr();
  const int64_t k = codes.size(codes.dim() - 1);
  Py_BEGIN_ALLOW_THREADS
  st = rw4_int8_dequantize(cp, sp, m, k, op, code, c.stream);
  Py_END_ALLOW_THREADS
  return st == RW4_OK ? THPVariable_Wrap(out) : none();
  END_HANDLE_TH_ERRORS
}

// int8_linear(codes, scale, weight, weight_scale, bias or None, residual or None, dtype)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !plain(a[0], -1) || !THPDtype_Check(a[6])) return none();
  const at::Tensor& codes = THPVariable_Unpack(a[0]);
  const at::ScalarType dt = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int dev = codes.get_device(), code = dtype_code(dt);
  int64_t m, wrows;
  Call c;
  if (code < 0 || !codes_ok(codes, a[1], dev, m) || !plain(a[2], dev) || !here(dev, c))
    return none();
  const at::Tensor& w = THPVariable_Unpack(a[2]);
  if (w.dim() != 2 || !codes_ok(w, a[3], dev, wrows)) return none();
  const int64_t k = codes.size(codes.dim() - 1), rows = w.size(0);
  if (w.size(1) != k) return none();
  const void *bias = nullptr, *residual = nullptr;
  if (a[4] != Py_None) {
    if (!plain(a[4], dev)) return none();
    const at::Tensor& b = THPVariable_Unpack(a[4]);
    if (b.scalar_type() != dt || b.dim() != 1 || b.size(0) != rows || !b.is_contiguous())
      return none();
    bias = b.const_data_ptr();
  }
  c10::SmallVector<int64_t, 6> shape(codes.sizes().begin(), codes.sizes().end());
  shape.back() = rows;
  if (a[5] != Py_None) {
    if (!plain(a[5], dev)) return none();
    const at::Tensor& r = THPVariable_Unpack(a[5]);
    if (r.scalar_type() != dt || r.sizes() != at::IntArrayRef(shape) || !r.is_contiguous())
      return none();
    residual = r.const_data_ptr();
  }
  at::Tensor out = empty(shape, dt, codes.device());
  int st;
  const int8_t* cp = static_cast<const int8_t*>(codes.const_data_ptr());
  const float* sp = static_cast<const float*>(THPVariable_Unpack(a[1]).const_data_ptr());
  const int8_t* wp = static_cast<const int8_t*>(w.const_data_ptr());
  const float* wsp = static_cast<const float*>(THPVariable_Unpack(a[3]).const_data_ptr());
  void* op = out.mutable_data_ptr();
  Py_BEGIN_ALLOW_THREADS
  st = rw4_int8_linear(cp, sp, m, k, wp, wsp, rows, bias, residual, op, code, 0, c.stream);
  Py_END_ALLOW_THREADS
  return st == RW4_OK ? THPVariable_Wrap(out) : none();
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef kMethods[] = {
    {"int8_quantize", fast<quantize>(), METH_FASTCALL, "(x, gate)"},
    {"int8_rmsnorm", fast<rmsnorm>(), METH_FASTCALL, "(x, weight, eps, residual)"},
    {"int8_dequantize", fast<dequantize>(), METH_FASTCALL, "(codes, scale, dtype)"},
    {"int8_linear", fast<linear>(), METH_FASTCALL,
     "(codes, scale, weight, weight_scale, bias, residual, dtype)"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_rw4_native",
                       "Host fast path of the 8-bit operators.", -1, kMethods};

}  // namespace

// `torch_version`: what this was compiled against; kernels.py takes it beside that torch alone.
PyMODINIT_FUNC PyInit__rw4_native() {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "torch_version", RW4_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
