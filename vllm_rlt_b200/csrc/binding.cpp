// Direct Python entry of the projection operators: argument checks, output
// allocation and the C call in one step. A decode step calls them several
// times per layer at sizes that take the GPU 5 to 10 microseconds; through
// ctypes the host needed 10 microseconds a call, here about 5.
//
// Every refusal is a ValueError made before any launch, the tensors' device
// last, so that the other checks can be met by tensors of any device.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "rlt_b200.h"

namespace {

PyObject* g_check = nullptr;  // callable: (return code, what) -> raises

struct PyError {};  // a Python exception is set

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": ", name, " must be a tensor");
  return THPVariable_Unpack(o);
}

// The tensor, or NULL for None.
const at::Tensor* optional(PyObject* o, const char* what, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, what, name);
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RLT_F32;
    case at::kHalf: return RLT_F16;
    case at::kBFloat16: return RLT_BF16;
    default: return -1;
  }
}

int32_t int32_size(int64_t n, const char* what) {
  // numbers as text: one streamed into the message ended the process here
  TORCH_CHECK_VALUE(n <= RLT_PROJ_MAX_SIZE, what, ": sizes must be at most ",
                    std::to_string(RLT_PROJ_MAX_SIZE));
  return static_cast<int32_t>(n);
}

// A lazily negated tensor (the imaginary part of a conjugate view) holds the
// opposite of its values, and one of lazy zeros holds none.
void holds_values(const at::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(!t.is_neg() && !t._is_zerotensor(), what,
                    ": a tensor does not hold its values (resolve_neg, clone)");
}

struct Operands {
  at::Tensor x;  // rows of contiguous features
  int32_t rows, inner, outer, dtype;
  int64_t x_rs, w_ns, w_ks;
};

Operands operands(const at::Tensor& x, const at::Tensor& w, const char* what) {
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1), what,
                    ": expected x [rows, in] and weight [out, in]");
  Operands o;
  o.dtype = dtype_code(x.scalar_type());
  TORCH_CHECK_VALUE(o.dtype >= 0 && w.scalar_type() == x.scalar_type(), what,
                    ": x and weight must share a float32, float16 or bfloat16 dtype");
  TORCH_CHECK_VALUE(w.device() == x.device(), what, ": all tensors must live on the same device");
  TORCH_CHECK_VALUE(x.layout() == at::kStrided && w.layout() == at::kStrided, what,
                    ": tensors must be dense");
  holds_values(x, what);
  holds_values(w, what);
  TORCH_CHECK_VALUE(x.size(1) > 0, what, ": in_features must be positive");
  o.rows = int32_size(x.size(0), what);
  o.inner = int32_size(x.size(1), what);
  o.outer = int32_size(w.size(0), what);
  o.w_ns = w.stride(0);
  o.w_ks = w.stride(1);
  if (o.w_ks == 1 || o.inner == 1) {
    o.w_ks = 1;
  } else {
    TORCH_CHECK_VALUE(o.w_ns == 1 || o.outer == 1, what,
                      ": one dimension of weight must be contiguous");
    o.w_ns = 1;
  }
  o.x = x;
  return o;
}

void rows_like(const at::Tensor& t, int64_t outer, const Operands& o, const char* name,
               const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == o.rows && t.size(1) == outer &&
                        t.scalar_type() == o.x.scalar_type() && t.device() == o.x.device() &&
                        t.layout() == at::kStrided,
                    what, ": ", name, " must be [rows, out] of x's dtype and device");
  holds_values(t, what);
}

void check_output(const at::Tensor* out, int64_t outer, const Operands& o, const char* what) {
  if (out == nullptr) return;
  rows_like(*out, outer, o, "out", what);
  TORCH_CHECK_VALUE((outer <= 1 || out->stride(1) == 1) && (o.rows <= 1 || out->stride(0) >= outer),
                    what, ": rows of out must be contiguous and apart");
}

void on_cuda(Operands& o, const char* what) {
  TORCH_CHECK_VALUE(o.x.is_cuda(), what, " requires a CUDA device");
  if (o.x.stride(1) != 1) o.x = o.x.contiguous();
  o.x_rs = o.x.stride(0);
}

void checked(int rc, const char* what) {
  if (rc == RLT_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, what);
  Py_XDECREF(r);
  TORCH_CHECK(r == nullptr, what, ": error ", std::to_string(rc));
  throw PyError();
}

// The current device's.
int32_t* status_word(const char* what) {
  int32_t* word = nullptr;
  checked(rlt_status_word(&word), what);
  return word;
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  if (bytes == 0) return at::Tensor();
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int64_t whole(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyError();
  return v;
}

at::Tensor do_linear(PyObject* const* a) {
  const char* what = "linear";
  const at::Tensor& w = tensor(a[1], what, "weight");
  Operands o = operands(tensor(a[0], what, "x"), w, what);
  const at::Tensor* bias = optional(a[2], what, "bias");
  const int32_t act = static_cast<int32_t>(whole(a[3]));
  const at::Tensor* residual = optional(a[4], what, "residual");
  const at::Tensor* out = optional(a[5], what, "out");
  at::Tensor held_bias, held_residual, result;
  if (bias != nullptr) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == o.outer &&
                          bias->scalar_type() == o.x.scalar_type() &&
                          bias->device() == o.x.device() && bias->layout() == at::kStrided,
                      what, ": bias must be [out] of x's dtype and device");
    holds_values(*bias, what);
  }
  if (residual != nullptr) rows_like(*residual, o.outer, o, "residual", what);
  check_output(out, o.outer, o, what);
  on_cuda(o, what);
  c10::cuda::CUDAGuard guard(o.x.device());
  if (bias != nullptr) held_bias = bias->stride(0) == 1 ? *bias : bias->contiguous();
  if (residual != nullptr)
    held_residual = residual->stride(1) == 1 ? *residual : residual->contiguous();
  result = out != nullptr ? *out : at::empty({o.rows, o.outer}, o.x.options());
  if (o.rows == 0 || o.outer == 0) return result;
  int32_t* status = status_word(what);
  const size_t need = rlt_linear_workspace_bytes(o.x.data_ptr(), w.data_ptr(), o.dtype, o.rows,
                                                 o.inner, o.outer, 0, o.x_rs, o.w_ns, o.w_ks);
  const at::Tensor work = scratch(need, o.x);
  checked(rlt_linear(o.x.data_ptr(), w.data_ptr(), ptr(held_bias), ptr(held_residual),
                     result.data_ptr(), ptr(work), need, status, o.dtype, o.rows, o.inner, o.outer,
                     act, o.x_rs, o.w_ns, o.w_ks,
                     residual != nullptr ? held_residual.stride(0) : 0, result.stride(0),
                     c10::cuda::getCurrentCUDAStream().stream()),
          what);
  return result;
}

at::Tensor do_gated(PyObject* const* a) {
  const char* what = "gated linear";
  const at::Tensor& w = tensor(a[1], what, "weight");
  Operands o = operands(tensor(a[0], what, "x"), w, what);
  const int32_t act = static_cast<int32_t>(whole(a[2]));
  const at::Tensor* out = optional(a[3], what, "out");
  TORCH_CHECK_VALUE(o.outer % 2 == 0, what, ": weight must hold as many gate rows as up rows");
  const int32_t outer = o.outer / 2;
  check_output(out, outer, o, what);
  on_cuda(o, what);
  c10::cuda::CUDAGuard guard(o.x.device());
  at::Tensor result = out != nullptr ? *out : at::empty({o.rows, outer}, o.x.options());
  if (o.rows == 0 || outer == 0) return result;
  int32_t* status = status_word(what);
  const size_t need = rlt_linear_workspace_bytes(o.x.data_ptr(), w.data_ptr(), o.dtype, o.rows,
                                                 o.inner, outer, 1, o.x_rs, o.w_ns, o.w_ks);
  const at::Tensor work = scratch(need, o.x);
  checked(rlt_gated_linear(o.x.data_ptr(), w.data_ptr(), result.data_ptr(), ptr(work), need,
                           status, o.dtype, o.rows, o.inner, outer, act, o.x_rs, o.w_ns, o.w_ks,
                           result.stride(0), c10::cuda::getCurrentCUDAStream().stream()),
          what);
  return result;
}

// (chosen tokens where `tokens` is None, log-probabilities)
std::pair<at::Tensor, at::Tensor> do_head(PyObject* const* a) {
  const at::Tensor* tokens = a[2] == Py_None ? nullptr : &tensor(a[2], "token logprobs", "tokens");
  const char* what = tokens != nullptr ? "token logprobs" : "greedy tokens";
  const at::Tensor& w = tensor(a[1], what, "weight");
  Operands o = operands(tensor(a[0], what, "hidden"), w, what);
  TORCH_CHECK_VALUE(o.outer > 0, what, ": the vocabulary must not be empty");
  if (tokens != nullptr) {
    TORCH_CHECK_VALUE(tokens->dim() == 1 && tokens->scalar_type() == at::kLong &&
                          tokens->size(0) == o.rows && tokens->layout() == at::kStrided,
                      what, ": tokens must be int64 [rows]");
    TORCH_CHECK_VALUE(tokens->device() == o.x.device(), what,
                      ": all tensors must live on the same device");
  }
  on_cuda(o, what);
  c10::cuda::CUDAGuard guard(o.x.device());
  at::Tensor held, chosen;
  if (tokens != nullptr)
    held = tokens->contiguous();
  else
    chosen = at::empty({o.rows}, o.x.options().dtype(at::kLong));
  at::Tensor logprobs = at::empty({o.rows}, o.x.options().dtype(at::kFloat));
  if (o.rows == 0) return {chosen, logprobs};
  int32_t* status = status_word(what);
  const size_t need = rlt_vocab_head_workspace_bytes(o.x.data_ptr(), w.data_ptr(), o.dtype, o.rows,
                                                     o.inner, o.outer, o.x_rs, o.w_ns, o.w_ks);
  const at::Tensor work = scratch(need, o.x);
  checked(rlt_vocab_head(o.x.data_ptr(), w.data_ptr(), static_cast<const int64_t*>(ptr(held)),
                         static_cast<int64_t*>(ptr(chosen)),
                         static_cast<float*>(logprobs.data_ptr()), ptr(work), need, status,
                         o.dtype, o.rows, o.inner, o.outer, o.x_rs, o.w_ns, o.w_ks,
                         c10::cuda::getCurrentCUDAStream().stream()),
          what);
  return {chosen, logprobs};
}

bool arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 6)) return nullptr;
  try {
    return THPVariable_Wrap(do_linear(a));
  } catch (const PyError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_gated(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 4)) return nullptr;
  try {
    return THPVariable_Wrap(do_gated(a));
  } catch (const PyError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_head(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 3)) return nullptr;
  try {
    auto [chosen, logprobs] = do_head(a);
    if (!chosen.defined()) return THPVariable_Wrap(std::move(logprobs));
    PyObject* c = THPVariable_Wrap(std::move(chosen));
    PyObject* l = THPVariable_Wrap(std::move(logprobs));
    PyObject* both = c != nullptr && l != nullptr ? PyTuple_Pack(2, c, l) : nullptr;
    Py_XDECREF(c);
    Py_XDECREF(l);
    return both;
  } catch (const PyError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 1)) return nullptr;
  Py_INCREF(a[0]);
  Py_XSETREF(g_check, a[0]);
  Py_RETURN_NONE;
}

#define RLT_METHOD(name, fn, doc) \
  {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, doc}

PyMethodDef methods[] = {
    RLT_METHOD("setup", py_setup, "setup(check)"),
    RLT_METHOD("linear", py_linear, "linear(x, weight, bias, activation, residual, out)"),
    RLT_METHOD("gated_linear", py_gated, "gated_linear(x, weight, activation, out)"),
    RLT_METHOD("vocab_head", py_head, "vocab_head(hidden, weight, tokens)"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rlt_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__rlt_torch() { return PyModule_Create(&module); }
