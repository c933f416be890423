// Python entry points of the block-scaled 8-bit operators on torch tensors.
//
// The checks, output allocations and argument structs behind forgetune_b200/fp8.py
// in C++, ending in the C ABI (include/forgetune_b200.h).  A one-row call costs
// more on the host than on the GPU.  Host time per call on the GPU's machine,
// against the same steps in Python through ctypes: quantize_rows 5.1 us (9.2),
// rms_norm with residual and quantised output 6.1 (13.5), fp8_linear 4.4
// (8.3); about 1.3 us of it is each output's allocation, 2.7 the launch.
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

#include "forgetune_b200.h"

#ifndef FTB_TORCH_OPS_TARGET
#define FTB_TORCH_OPS_TARGET "unknown"
#endif
// Read from the file, before it is loaded: the layouts above are compiled in.
extern "C" __attribute__((used)) const char ftb_torch_ops_built_for[] = "_torch_ops built for: " FTB_TORCH_OPS_TARGET;

namespace {

PyObject* g_shape_error = nullptr;    // forgetune_b200.errors.InvalidShapeError
PyObject* g_runtime_error = nullptr;  // forgetune_b200.errors.ForgeTuneRuntimeError

struct Refused {
  PyObject* type;
  std::string what;
};
[[noreturn]] void type_error(const std::string& s) { throw Refused{PyExc_TypeError, s}; }
[[noreturn]] void value_error(const std::string& s) { throw Refused{PyExc_ValueError, s}; }
[[noreturn]] void shape_error(const std::string& s) { throw Refused{g_shape_error, s}; }

constexpr int64_t kBlock = 128;
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

std::string show(int64_t a, int64_t b) { return "(" + std::to_string(a) + ", " + std::to_string(b) + ")"; }
std::string show(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int plain_type(at::ScalarType t) {
  return t == at::kFloat ? FTB_F32 : t == at::kHalf ? FTB_F16 : t == at::kBFloat16 ? FTB_BF16 : -1;
}

// Row stride of a matrix whose rows are contiguous and do not overlap, or -1.
int64_t row_stride(const at::Tensor& t) {
  const int64_t rows = t.size(0), cols = t.size(1);
  if (cols > 1 && t.stride(1) != 1) return -1;
  if (rows <= 1) return cols;
  return t.stride(0) >= cols ? t.stride(0) : -1;
}

// The same of 8-bit rows, which also start on multiples of `unit` bytes.
int64_t row_stride8(const at::Tensor& t, int64_t unit) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % unit) return -1;
  const int64_t ld = row_stride(t);
  if (ld < 0) return -1;
  if (t.size(0) <= 1) return (ld + unit - 1) / unit * unit;
  return ld % unit ? -1 : ld;
}

struct Matrix {
  at::Tensor t;
  ftb_matrix a{nullptr, 0, 0};
  int64_t m = 0, k = 0;
};

ftb_matrix as_matrix(const at::Tensor& t, int64_t ld) { return {t.data_ptr(), ld, plain_type(t.scalar_type())}; }

// A forward-mode tangent would be dropped, which reads as a derivative of zero.
void check_tangent(const at::Tensor& t, const char* what) {
  if (t._fw_grad(0).defined())
    value_error(std::string(what) + " has a forward-mode tangent: the operators have no derivatives (unpack it first)");
}

// A plain 2-D CUDA input, copied where its rows are not contiguous.
Matrix input(PyObject* o, const char* what) {
  const at::Tensor* t = tensor(o);
  if (!t || !t->is_cuda() || plain_type(t->scalar_type()) < 0 || t->layout() != at::kStrided)
    type_error(std::string(what) + " must be a float32, float16 or bfloat16 CUDA tensor");
  if (t->dim() != 2 || t->size(1) < 1)
    shape_error(std::string(what) + " must be 2-D with at least one column, got " + show(t->sizes()));
  check_tangent(*t, what);
  Matrix r;
  r.m = t->size(0);
  r.k = t->size(1);
  r.t = t->is_neg() ? t->resolve_neg() : *t;  // a view that stands for the negated values
  int64_t ld = row_stride(r.t);
  if (ld < 0) {
    r.t = r.t.contiguous();
    ld = r.k;
  }
  r.a = as_matrix(r.t, ld);
  return r;
}

// A caller's output is written past autograd: refused where autograd would
// have to know, as torch's own out= forms do (a leaf in no_grad is fine).
void check_written(const at::Tensor& t, const char* what) {
  check_tangent(t, what);
  if (t.requires_grad() && at::GradMode::is_enabled())
    value_error(std::string(what) + " requires grad: the operators have no backward pass (call them in torch.no_grad())");
}

// ... and counted as a change in place, so that a backward pass that saved the
// old values refuses to run on the new ones.  Tensors made in inference mode
// have no count.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_place(const at::Tensor& t, const char* what, int64_t m, int64_t n, at::Device dev) {
  if (t.dim() != 2 || t.size(0) != m || t.size(1) != n)
    shape_error(std::string(what) + " must be " + show(m, n) + ", got " + show(t.sizes()));
  if (t.device() != dev)
    value_error(std::string(what) + " is on " + t.device().str() + ", the input on " + dev.str());
}

// A new plain output, or the caller's.
Matrix output(PyObject* o, const char* what, int64_t m, int64_t n, at::ScalarType type, at::Device dev) {
  Matrix r;
  r.m = m;
  r.k = n;
  if (o == Py_None) {
    r.t = at::empty_strided({m, n}, {n, 1}, at::TensorOptions().dtype(type).device(dev));
    r.a = as_matrix(r.t, n);
    return r;
  }
  const at::Tensor* t = tensor(o);
  if (!t || t->scalar_type() != type || t->layout() != at::kStrided || t->is_neg())
    type_error(std::string(what) + " must be a " + c10::toString(type) + " tensor");
  check_place(*t, what, m, n, dev);
  const int64_t ld = row_stride(*t);
  if (ld < 0) shape_error(std::string(what) + ": rows must be contiguous and must not overlap");
  check_written(*t, what);
  r.t = *t;
  r.a = as_matrix(r.t, ld);
  return r;
}

struct Fp8 {
  at::Tensor data, scales;
  ftb_fp8_matrix a{nullptr, 0, nullptr, 0};
  int64_t m = 0, k = 0;
};

// 8-bit values [m, k] with their scales; `row_block`: 1 (rows) or 128 (a weight).
Fp8 fp8(PyObject* data, PyObject* scales, int64_t row_block, const char* what) {
  const at::Tensor *d = tensor(data), *s = tensor(scales);
  if (!d || d->scalar_type() != at::kFloat8_e4m3fn || d->layout() != at::kStrided)
    type_error(std::string(what) + ": data must be a torch.float8_e4m3fn tensor");
  if (!s || s->scalar_type() != at::kFloat8_e8m0fnu || s->layout() != at::kStrided)
    type_error(std::string(what) + ": scales must be a torch.float8_e8m0fnu tensor");
  if (d->is_neg() || s->is_neg()) type_error(std::string(what) + ": data and scales must not be negated views");
  if (d->dim() != 2 || d->size(1) < 1)
    shape_error(std::string(what) + ": data must be [rows, k] with k >= 1, got " + show(d->sizes()));
  Fp8 r;
  r.m = d->size(0);
  r.k = d->size(1);
  const int64_t rows = (r.m + row_block - 1) / row_block;
  if (s->dim() != 2 || s->size(0) != rows || s->size(1) != blocks(r.k))
    shape_error(std::string(what) + ": scales of data " + show(r.m, r.k) + " must be " + show(rows, blocks(r.k)) +
                ", got " + show(s->sizes()));
  if (d->device() != s->device()) value_error(std::string(what) + ": data and scales are on different devices");
  r.data = *d;
  r.scales = *s;
  return r;
}

// ... in the layout that the operators take.
void lay_out(Fp8& r, const char* what) {
  const int64_t ld = row_stride8(r.data, 16), s_ld = row_stride8(r.scales, 4);
  if (ld < 0 || s_ld < 0)
    shape_error(std::string(what) + ": rows of data must start on 16-byte and rows of scales on 4-byte boundaries "
                                    "(see pack)");
  r.a = {static_cast<uint8_t*>(r.data.data_ptr()), ld, static_cast<uint8_t*>(r.scales.data_ptr()), s_ld};
}

Fp8 new_fp8(int64_t m, int64_t k, int64_t row_block, at::Device dev) {
  Fp8 r;
  const int64_t ld = (k + 15) / 16 * 16, kb = blocks(k), s_ld = (kb + 3) / 4 * 4;
  r.data = at::empty_strided({m, k}, {ld, 1}, at::TensorOptions().dtype(at::kFloat8_e4m3fn).device(dev));
  r.scales = at::empty_strided({(m + row_block - 1) / row_block, kb}, {s_ld, 1},
                               at::TensorOptions().dtype(at::kFloat8_e8m0fnu).device(dev));
  r.m = m;
  r.k = k;
  r.a = {static_cast<uint8_t*>(r.data.data_ptr()), ld, static_cast<uint8_t*>(r.scales.data_ptr()), s_ld};
  return r;
}

// A new quantised output, or the caller's.
Fp8 fp8_output(PyObject* data, PyObject* scales, const char* what, int64_t m, int64_t k, at::Device dev) {
  if (data == Py_None) return new_fp8(m, k, 1, dev);
  Fp8 r = fp8(data, scales, 1, what);
  check_place(r.data, what, m, k, dev);
  check_written(r.data, what);
  check_written(r.scales, what);
  lay_out(r, what);
  return r;
}

// A float32 vector of n values, or none.
at::Tensor vector(PyObject* o, const char* what, int64_t n, at::Device dev) {
  if (o == Py_None) return at::Tensor();
  const at::Tensor* t = tensor(o);
  if (!t || t->scalar_type() != at::kFloat || t->layout() != at::kStrided)
    type_error(std::string(what) + " must be a float32 tensor");
  if (t->dim() != 1 || t->size(0) != n)
    shape_error(std::string(what) + " must be [" + std::to_string(n) + "], got " + show(t->sizes()));
  if (t->device() != dev)
    value_error(std::string(what) + " is on " + t->device().str() + ", the input on " + dev.str());
  check_tangent(*t, what);
  const at::Tensor v = t->is_neg() ? t->resolve_neg() : *t;
  return n == 1 || v.stride(0) == 1 ? v : v.contiguous();
}

// One C call on the current stream of `dev`.
template <typename Args>
void call(const char* name, int (*fn)(const Args*, void*), const Args& args, at::Device dev) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev.index()) guard.set_device(dev);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(&args, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0)
    throw Refused{g_runtime_error, std::string(name) + " failed (" + std::to_string(rc) + "): " + ftb_last_error()};
}

// The caller's outputs among these (`given`: what the caller passed, None for a new tensor).
void written(PyObject* given, const Matrix& y) {
  if (given != Py_None) written(y.t);
}
void written(PyObject* given, const Fp8& q) {
  if (given == Py_None) return;
  written(q.data);
  written(q.scales);
}

void run_quantize_rows(const Matrix& x, const Fp8& q) {
  ftb_quantize_args a{x.a, q.a, x.m, x.k};
  call("ftb_quantize_rows", ftb_quantize_rows, a, x.t.device());
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused{nullptr, ""};
  return v != 0;
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair(PyObject* a, PyObject* b) {
  if (!a || !b) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyObject* r = PyTuple_Pack(2, a, b);
  Py_DECREF(a);
  Py_DECREF(b);
  return r;
}
PyObject* none() { Py_RETURN_NONE; }

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& body) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return nullptr;
  }
  try {
    return body();
  } catch (const Refused& r) {
    if (r.type) PyErr_SetString(r.type, r.what.c_str());
  } catch (...) {  // torch's own: out of memory and the like
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// check(data, scales, row_block, name) -> whether both are laid out for the operators
PyObject* op_check(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const char* name = PyUnicode_AsUTF8(a[3]);
    if (!name) return nullptr;
    const Fp8 r = fp8(a[0], a[1], PyLong_AsLongLong(a[2]), name);
    return PyBool_FromLong(row_stride8(r.data, 16) >= 0 && row_stride8(r.scales, 4) >= 0);
  });
}

// quantize_rows(x, out data, out scales) -> (data, scales)
PyObject* op_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    const Matrix x = input(a[0], "quantize_rows: x");
    const Fp8 q = fp8_output(a[1], a[2], "quantize_rows: out", x.m, x.k, x.t.device());
    run_quantize_rows(x, q);
    written(a[1], q);
    return pair(wrap(q.data), wrap(q.scales));
  });
}

// quantize_weight(w) -> (data, scales)
PyObject* op_quantize_weight(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 1, [&]() -> PyObject* {
    const Matrix w = input(a[0], "quantize_weight: w");
    if (w.m < 1) shape_error("quantize_weight: w must have at least one row");
    const Fp8 q = new_fp8(w.m, w.k, kBlock, w.t.device());
    ftb_quantize_args args{w.a, q.a, w.m, w.k};
    call("ftb_quantize_weight", ftb_quantize_weight, args, w.t.device());
    return pair(wrap(q.data), wrap(q.scales));
  });
}

// rms_norm(x, weight, eps, residual, quantize, out (data), out scales, residual_out)
//   -> (y or data, scales or None, h or None)
PyObject* op_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Matrix x = input(a[0], "rms_norm: x");
    const at::Device dev = x.t.device();
    const at::ScalarType type = x.t.scalar_type();
    const at::Tensor weight = vector(a[1], "rms_norm: weight", x.k, dev);
    const double eps = PyFloat_AsDouble(a[2]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    ftb_rms_norm_args args{};
    args.x = x.a;
    args.weight = weight.defined() ? static_cast<const float*>(weight.data_ptr()) : nullptr;
    args.eps = eps;
    args.m = x.m;
    args.k = x.k;
    Matrix res, h, y;
    Fp8 q;
    if (a[3] != Py_None) {
      res = input(a[3], "rms_norm: residual");
      if (res.t.scalar_type() != type)
        type_error(std::string("rms_norm: residual must be ") + c10::toString(type) + ", got " +
                   c10::toString(res.t.scalar_type()));
      check_place(res.t, "rms_norm: residual", x.m, x.k, dev);
      h = output(a[7], "rms_norm: residual_out", x.m, x.k, type, dev);
      args.residual = res.a;
      args.h = h.a;
    } else if (a[7] != Py_None) {
      value_error("rms_norm: residual_out needs a residual");
    }
    const bool quantize = truth(a[4]);
    if (quantize) {
      q = fp8_output(a[5], a[6], "rms_norm: out", x.m, x.k, dev);
      args.q = q.a;
    } else {
      y = output(a[5], "rms_norm: out", x.m, x.k, type, dev);
      args.y = y.a;
    }
    call("ftb_rms_norm", ftb_rms_norm, args, dev);
    if (quantize) written(a[5], q);
    else written(a[5], y);
    if (h.t.defined()) written(a[7], h);
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, wrap(quantize ? q.data : y.t));
    PyTuple_SET_ITEM(r, 1, quantize ? wrap(q.scales) : none());
    PyTuple_SET_ITEM(r, 2, a[3] != Py_None ? wrap(h.t) : none());
    return r;
  });
}

// linear(x (data), x scales or None for a plain x, w data, w scales, bias, relu, residual, out_dtype, quantize,
//        out (data), out scales) -> (y or data, scales or None)
PyObject* op_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const bool quantize = truth(a[8]);
    at::ScalarType type = at::kFloat;
    bool typed = a[7] != Py_None;
    if (typed) {
      if (quantize) value_error("fp8_linear: a quantised result has no out_dtype");
      if (THPDtype_Check(a[7])) type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
      if (!THPDtype_Check(a[7]) || plain_type(type) < 0)
        type_error("fp8_linear: out_dtype must be float32, float16 or bfloat16");
    }
    Matrix plain;
    Fp8 x;
    if (a[1] == Py_None) {
      plain = input(a[0], "fp8_linear: x");
      if (!typed) type = plain.t.scalar_type(), typed = true;
      x.m = plain.m;
      x.k = plain.k;
    } else {
      x = fp8(a[0], a[1], 1, "fp8_linear: x");
      if (!x.data.is_cuda()) type_error("fp8_linear: x must be on a CUDA device");
      lay_out(x, "fp8_linear: x");
    }
    const at::Device dev = plain.t.defined() ? plain.t.device() : x.data.device();
    Fp8 w = fp8(a[2], a[3], kBlock, "fp8_linear: weight");
    if (w.k != x.k)
      shape_error("fp8_linear: x is " + show(x.m, x.k) + ", weight " + show(w.m, w.k) + ": their depths differ");
    if (w.data.device() != dev)
      value_error("fp8_linear: weight is on " + w.data.device().str() + ", the input on " + dev.str());
    lay_out(w, "fp8_linear: weight");
    const int64_t m = x.m, nn = w.m;
    const at::Tensor bias = vector(a[4], "fp8_linear: bias", nn, dev);
    ftb_fp8_linear_args args{};
    args.bias = bias.defined() ? static_cast<const float*>(bias.data_ptr()) : nullptr;
    Matrix res, y;
    Fp8 q;
    if (a[6] != Py_None) {
      res = input(a[6], "fp8_linear: residual");
      check_place(res.t, "fp8_linear: residual", m, nn, dev);
      args.residual = res.a;
      if (!typed) type = res.t.scalar_type();
    }
    if (quantize) {
      q = fp8_output(a[9], a[10], "fp8_linear: out", m, nn, dev);
      args.q = q.a;
    } else {
      y = output(a[9], "fp8_linear: out", m, nn, type, dev);
      args.y = y.a;
    }
    args.m = m;
    args.n = nn;
    args.k = x.k;
    args.flags = truth(a[5]) ? FTB_FP8_RELU : 0;
    if (plain.t.defined()) {
      x = new_fp8(m, plain.k, 1, dev);
      run_quantize_rows(plain, x);
    }
    args.a = x.a;
    args.w = w.a;
    call("ftb_fp8_linear", ftb_fp8_linear, args, dev);
    if (quantize) written(a[9], q);
    else written(a[9], y);
    return pair(wrap(quantize ? q.data : y.t), quantize ? wrap(q.scales) : none());
  });
}

PyMethodDef kMethods[] = {
    {"check", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_check)), METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_quantize_rows)), METH_FASTCALL, nullptr},
    {"quantize_weight", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_quantize_weight)), METH_FASTCALL,
     nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_rms_norm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() {
  PyObject* errors = PyImport_ImportModule("forgetune_b200.errors");
  if (!errors) return nullptr;
  g_shape_error = PyObject_GetAttrString(errors, "InvalidShapeError");
  g_runtime_error = PyObject_GetAttrString(errors, "ForgeTuneRuntimeError");
  Py_DECREF(errors);
  if (!g_shape_error || !g_runtime_error) return nullptr;
  return PyModule_Create(&kModule);
}
