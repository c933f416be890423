// Python entry points of the operators on torch tensors.
//
// The checks, output allocations and argument structs behind forgetune_b200/fp8.py
// and decoder.py in C++, ending in the C ABI (include/forgetune_b200.h).  A one-row call costs
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

#include <cmath>
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

// ---------------------------------------------------------------------------
// a decoder layer's heads, paged cache and logits (decoder.py)
// ---------------------------------------------------------------------------
struct Heads {
  at::Tensor t;
  ftb_heads a{nullptr, 0, 0, 0};
  int64_t tokens = 0, heads = 0, dim = 0;
};

// Strides of [tokens, heads, dim] whose heads are whole and apart; false for others.
bool lay_heads(Heads& r) {
  const at::Tensor& t = r.t;
  r.tokens = t.size(0);
  r.heads = t.size(1);
  r.dim = t.size(2);
  const int64_t token = r.tokens > 1 ? t.stride(0) : 0, head = r.heads > 1 ? t.stride(1) : 0;
  r.a = {t.data_ptr(), token, head, plain_type(t.scalar_type())};
  if (r.dim > 1 && t.stride(2) != 1) return false;
  if (r.tokens > 1 && r.heads > 1) {
    return token >= head ? head >= r.dim && token >= (r.heads - 1) * head + r.dim
                         : token >= r.dim && head >= (r.tokens - 1) * token + r.dim;
  }
  return (r.tokens <= 1 || token >= r.dim) && (r.heads <= 1 || head >= r.dim);
}

// A CUDA input of heads, copied where they are not whole or overlap.
Heads heads_input(PyObject* o, const char* what) {
  const at::Tensor* t = tensor(o);
  if (!t || !t->is_cuda() || plain_type(t->scalar_type()) < 0 || t->layout() != at::kStrided)
    type_error(std::string(what) + " must be a float32, float16 or bfloat16 CUDA tensor");
  if (t->dim() != 3 || t->size(1) < 1 || t->size(2) < 1)
    shape_error(std::string(what) + " must be [tokens, heads, dim] with at least one head and element, got " +
                show(t->sizes()));
  check_tangent(*t, what);
  Heads r;
  r.t = t->is_neg() ? t->resolve_neg() : *t;
  if (!lay_heads(r)) {
    r.t = r.t.contiguous();
    lay_heads(r);
  }
  return r;
}

void check_device(const at::Tensor& t, const char* what, at::Device dev) {
  if (t.device() != dev)
    value_error(std::string(what) + " is on " + t.device().str() + ", the input on " + dev.str());
}

void check_heads(const Heads& x, const char* what, int64_t tokens, int64_t dim, at::ScalarType type, at::Device dev) {
  if (x.tokens != tokens || x.dim != dim)
    shape_error(std::string(what) + " must be [" + std::to_string(tokens) + ", heads, " + std::to_string(dim) +
                "], got " + show(x.t.sizes()));
  if (x.t.scalar_type() != type) type_error(std::string(what) + " must be " + c10::toString(type));
  check_device(x.t, what, dev);
}

// New heads, or the caller's.
Heads heads_output(PyObject* o, const char* what, const Heads& like, at::ScalarType type) {
  Heads r;
  if (o == Py_None) {
    r.t = at::empty_strided({like.tokens, like.heads, like.dim}, {like.heads * like.dim, like.dim, 1},
                            at::TensorOptions().dtype(type).device(like.t.device()));
    lay_heads(r);
    return r;
  }
  const at::Tensor* t = tensor(o);
  if (!t || t->scalar_type() != type || t->layout() != at::kStrided || t->is_neg())
    type_error(std::string(what) + " must be a " + c10::toString(type) + " tensor");
  if (t->dim() != 3 || t->size(0) != like.tokens || t->size(1) != like.heads || t->size(2) != like.dim)
    shape_error(std::string(what) + " must be " + show(like.t.sizes()) + ", got " + show(t->sizes()));
  check_device(*t, what, like.t.device());
  r.t = *t;
  if (!lay_heads(r)) shape_error(std::string(what) + ": heads must be contiguous and must not overlap");
  check_written(*t, what);
  return r;
}

// Whole numbers on the device, copied where they are not in rows.
at::Tensor whole(PyObject* o, const char* what, int64_t dims, bool wide, at::Device dev) {
  const at::Tensor* t = tensor(o);
  if (!t || t->layout() != at::kStrided || !(t->scalar_type() == at::kInt || (wide && t->scalar_type() == at::kLong)))
    type_error(std::string(what) + " must be an int32 " + (wide ? "or int64 " : "") + "tensor");
  if (t->dim() != dims) shape_error(std::string(what) + " must be " + std::to_string(dims) + "-D, got " + show(t->sizes()));
  check_device(*t, what, dev);
  const bool rows = dims == 2 ? row_stride(*t) >= 0 : t->size(0) <= 1 || t->stride(0) == 1;
  return rows ? *t : t->contiguous();
}

struct Paged {
  at::Tensor keys, values, table, starts, lengths;
  ftb_paged_cache cache{};
  ftb_paged_batch batch{};
};

// The pools of keys and values, taken as they lie, and the batch.
Paged paged(const char* fn, PyObject* const* a, bool written_to, at::Device dev) {
  Paged r;
  at::Tensor* pool[2] = {&r.keys, &r.values};
  const char* names[2] = {": keys", ": values"};
  for (int i = 0; i < 2; ++i) {
    const std::string what = std::string(fn) + names[i];
    const at::Tensor* t = tensor(a[i]);
    if (!t || plain_type(t->scalar_type()) < 0 || t->layout() != at::kStrided || t->is_neg())
      type_error(what + " must be a float32, float16 or bfloat16 tensor");
    if (t->dim() != 4 || t->numel() == 0)
      shape_error(what + " must be [pages, page_size, kv_heads, dim], none of them 0, got " + show(t->sizes()));
    if (t->size(3) > 1 && t->stride(3) != 1) shape_error(what + ": the values of a head must be contiguous");
    check_device(*t, what.c_str(), dev);
    if (written_to) check_written(*t, what.c_str());
    else check_tangent(*t, what.c_str());
    *pool[i] = *t;
  }
  if (r.keys.sizes() != r.values.sizes())
    shape_error(std::string(fn) + ": values must be " + show(r.keys.sizes()) + " as keys are, got " + show(r.values.sizes()));
  if (r.keys.scalar_type() != r.values.scalar_type())
    type_error(std::string(fn) + ": values must be " + c10::toString(r.keys.scalar_type()) + " as keys are");
  auto stride = [](const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
  r.cache = {r.keys.data_ptr(), r.values.data_ptr(), stride(r.keys, 0), stride(r.keys, 1), stride(r.keys, 2),
             stride(r.values, 0), stride(r.values, 1), stride(r.values, 2), plain_type(r.keys.scalar_type()),
             r.keys.size(0), r.keys.size(1), r.keys.size(2), r.keys.size(3)};
  r.table = whole(a[2], (std::string(fn) + ": page_table").c_str(), 2, false, dev);
  r.starts = whole(a[3], (std::string(fn) + ": starts").c_str(), 1, false, dev);
  r.lengths = whole(a[4], (std::string(fn) + ": lengths").c_str(), 1, false, dev);
  const int64_t b = r.lengths.size(0);
  if (b < 1 || r.table.size(0) != b || r.table.size(1) < 1 || r.starts.size(0) != b + 1)
    shape_error(std::string(fn) + ": page_table must be [sequences, pages], starts [sequences + 1] and lengths "
                                  "[sequences], got " + show(r.table.sizes()) + ", " + show(r.starts.sizes()) + " and " +
                show(r.lengths.sizes()));
  r.batch = {static_cast<const int32_t*>(r.table.data_ptr()), row_stride(r.table), r.table.size(1), b,
             static_cast<const int32_t*>(r.starts.data_ptr()), static_cast<const int32_t*>(r.lengths.data_ptr())};
  return r;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}

struct Rotation {
  at::Tensor frequencies;
  ftb_rotation a{};
};

// frequencies (None: no rotation), eps, norm, interleaved, amplitude
Rotation rotation(const char* fn, PyObject* f, PyObject* const* a, int64_t dim, at::Device dev) {
  Rotation r;
  if (f != Py_None) {
    const std::string what = std::string(fn) + ": frequencies";
    const at::Tensor* t = tensor(f);
    if (!t || t->scalar_type() != at::kDouble || t->layout() != at::kStrided || t->is_neg())
      type_error(what + " must be a float64 tensor (see rope_frequencies)");
    if (t->dim() != 1 || t->size(0) < 1 || 2 * t->size(0) > dim)
      shape_error(what + " must be [pairs] with at most half of dim " + std::to_string(dim) + ", got " + show(t->sizes()));
    check_device(*t, what.c_str(), dev);
    check_tangent(*t, what.c_str());
    r.frequencies = t->size(0) == 1 || t->stride(0) == 1 ? *t : t->contiguous();
    r.a.frequencies = static_cast<const double*>(r.frequencies.data_ptr());
    r.a.pairs = t->size(0);
  }
  r.a.eps = number(a[0]);
  r.a.norm = truth(a[1]);
  r.a.interleaved = truth(a[2]);
  r.a.amplitude = number(a[3]);
  return r;
}

const float* head_weight(at::Tensor& keep, PyObject* o, const char* what, bool norm, int64_t dim, at::Device dev) {
  if (o != Py_None && !norm) value_error(std::string(what) + " needs norm=True");
  keep = vector(o, what, dim, dev);
  return keep.defined() ? static_cast<const float*>(keep.data_ptr()) : nullptr;
}

// rotate_heads(x, positions, frequencies, weight, eps, norm, interleaved, amplitude, out) -> y
PyObject* op_rotate_heads(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const Heads x = heads_input(a[0], "rotate_heads: x");
    const at::Device dev = x.t.device();
    const at::Tensor positions = whole(a[1], "rotate_heads: positions", 1, true, dev);
    if (positions.size(0) != x.tokens)
      shape_error("rotate_heads: positions must be [" + std::to_string(x.tokens) + "], got " + show(positions.sizes()));
    const Rotation rot = rotation("rotate_heads", a[2], a + 4, x.dim, dev);
    at::Tensor weight;
    ftb_rotate_args args{};
    args.weight = head_weight(weight, a[3], "rotate_heads: weight", rot.a.norm, x.dim, dev);
    const Heads y = heads_output(a[8], "rotate_heads: out", x, x.t.scalar_type());
    args.x = x.a;
    args.y = y.a;
    args.tokens = x.tokens;
    args.heads = x.heads;
    args.dim = x.dim;
    args.positions = positions.data_ptr();
    args.positions64 = positions.scalar_type() == at::kLong;
    args.rotation = rot.a;
    if (x.tokens > 0) call("ftb_rotate_heads", ftb_rotate_heads, args, dev);
    if (a[8] != Py_None) written(y.t);
    return wrap(y.t);
  });
}

// append_heads(q, k, v, keys, values, page_table, starts, lengths, frequencies, q_weight, k_weight, eps, norm,
//              interleaved, amplitude, out) -> q
PyObject* op_append_heads(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const Heads q = heads_input(a[0], "append_heads: q");
    const at::Device dev = q.t.device();
    const Heads k = heads_input(a[1], "append_heads: k"), v = heads_input(a[2], "append_heads: v");
    const Paged p = paged("append_heads", a + 3, true, dev);
    const at::ScalarType held = p.keys.scalar_type();
    check_heads(q, "append_heads: q", q.tokens, p.cache.dim, q.t.scalar_type(), dev);
    check_heads(k, "append_heads: k", q.tokens, p.cache.dim, q.t.scalar_type(), dev);
    check_heads(v, "append_heads: v", q.tokens, p.cache.dim, q.t.scalar_type(), dev);
    if (k.heads != p.cache.kv_heads || v.heads != p.cache.kv_heads)
      shape_error("append_heads: k and v must have the cache's " + std::to_string(p.cache.kv_heads) + " heads, got " +
                  std::to_string(k.heads) + " and " + std::to_string(v.heads));
    if (q.t.scalar_type() != held && q.t.scalar_type() != at::kFloat)
      type_error(std::string("append_heads: q, k and v must be float32 or the cache's ") + c10::toString(held));
    const Rotation rot = rotation("append_heads", a[8], a + 11, q.dim, dev);
    at::Tensor wq, wk;
    ftb_append_args args{};
    args.q_weight = head_weight(wq, a[9], "append_heads: q_weight", rot.a.norm, q.dim, dev);
    args.k_weight = head_weight(wk, a[10], "append_heads: k_weight", rot.a.norm, q.dim, dev);
    const Heads y = heads_output(a[15], "append_heads: out", q, held);
    args.q = q.a;
    args.k = k.a;
    args.v = v.a;
    args.q_out = y.a;
    args.tokens = q.tokens;
    args.heads = q.heads;
    args.cache = p.cache;
    args.batch = p.batch;
    args.rotation = rot.a;
    if (q.tokens > 0) call("ftb_append_heads", ftb_append_heads, args, dev);
    written(p.keys);
    written(p.values);
    if (a[15] != Py_None) written(y.t);
    return wrap(y.t);
  });
}

// paged_attention(q, keys, values, page_table, starts, lengths, scale, window, out) -> out
PyObject* op_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const Heads q = heads_input(a[0], "paged_attention: q");
    const at::Device dev = q.t.device();
    const Paged p = paged("paged_attention", a + 1, false, dev);
    check_heads(q, "paged_attention: q", q.tokens, p.cache.dim, p.keys.scalar_type(), dev);
    if (q.heads % p.cache.kv_heads)
      shape_error("paged_attention: q has " + std::to_string(q.heads) + " heads, the cache " +
                  std::to_string(p.cache.kv_heads) + ": not a multiple");
    ftb_attention_args args{};
    args.scale = a[6] == Py_None ? 1.0 / std::sqrt((double)q.dim) : number(a[6]);
    args.window = a[7] == Py_None ? 0 : integer(a[7]);
    if (args.window < 0) value_error("paged_attention: window must not be negative");
    const Heads y = heads_output(a[8], "paged_attention: out", q, q.t.scalar_type());
    args.q = q.a;
    args.out = y.a;
    args.tokens = q.tokens;
    args.heads = q.heads;
    args.cache = p.cache;
    args.batch = p.batch;
    if (q.tokens > 0) {
      c10::cuda::OptionalCUDAGuard guard;
      if (c10::cuda::current_device() != dev.index()) guard.set_device(dev);
      const int64_t bytes = ftb_paged_attention_workspace(&args);
      if (bytes < 0)
        throw Refused{g_runtime_error, "ftb_paged_attention_workspace failed (" + std::to_string(bytes) + "): " + ftb_last_error()};
      at::Tensor work;  // from torch's allocator: kept from other streams' use, and a graph's own under capture
      if (bytes > 0) {
        work = at::empty_strided({bytes}, {1}, at::TensorOptions().dtype(at::kByte).device(dev));
        args.workspace = work.data_ptr();
        args.workspace_bytes = bytes;
      }
      call("ftb_paged_attention", ftb_paged_attention, args, dev);
    }
    if (a[8] != Py_None) written(y.t);
    return wrap(y.t);
  });
}

// token_logprobs(logits, tokens, top) -> (logprobs, entropy[, top_logprobs, top_tokens])
PyObject* op_token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    const Matrix x = input(a[0], "token_logprobs: logits");
    const at::Device dev = x.t.device();
    const at::Tensor tokens = whole(a[1], "token_logprobs: tokens", 1, true, dev);
    if (tokens.size(0) != x.m)
      shape_error("token_logprobs: tokens must be [" + std::to_string(x.m) + "], got " + show(tokens.sizes()));
    const int64_t top = integer(a[2]);
    if (top < 0 || top > 64 || top > x.k)
      value_error("token_logprobs: top must be 0 to 64 and at most the " + std::to_string(x.k) + " logits of a row");
    auto make = [&](int64_t cols, at::ScalarType type) {
      const auto o = at::TensorOptions().dtype(type).device(dev);
      return cols ? at::empty_strided({x.m, cols}, {cols, 1}, o) : at::empty_strided({x.m}, {1}, o);
    };
    const at::Tensor logprobs = make(0, at::kFloat), entropy = make(0, at::kFloat);
    at::Tensor values, ids;
    ftb_logprobs_args args{};
    args.logits = x.a;
    args.m = x.m;
    args.n = x.k;
    args.tokens = tokens.data_ptr();
    args.tokens64 = tokens.scalar_type() == at::kLong;
    args.token_stride = 1;
    args.logprobs = static_cast<float*>(logprobs.data_ptr());
    args.entropy = static_cast<float*>(entropy.data_ptr());
    args.top = top;
    if (top) {
      values = make(top, at::kFloat);
      ids = make(top, at::kLong);
      args.top_logprobs = static_cast<float*>(values.data_ptr());
      args.top_tokens = static_cast<int64_t*>(ids.data_ptr());
    }
    if (x.m > 0) call("ftb_token_logprobs", ftb_token_logprobs, args, dev);
    PyObject* r = PyTuple_New(top ? 4 : 2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, wrap(logprobs));
    PyTuple_SET_ITEM(r, 1, wrap(entropy));
    if (top) {
      PyTuple_SET_ITEM(r, 2, wrap(values));
      PyTuple_SET_ITEM(r, 3, wrap(ids));
    }
    return r;
  });
}

PyMethodDef kMethods[] = {
    {"check", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_check)), METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_quantize_rows)), METH_FASTCALL, nullptr},
    {"quantize_weight", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_quantize_weight)), METH_FASTCALL,
     nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_rms_norm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_linear)), METH_FASTCALL, nullptr},
    {"rotate_heads", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_rotate_heads)), METH_FASTCALL, nullptr},
    {"append_heads", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_append_heads)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_paged_attention)), METH_FASTCALL,
     nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(op_token_logprobs)), METH_FASTCALL,
     nullptr},
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
