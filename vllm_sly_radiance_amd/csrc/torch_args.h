// What the bindings of this package's C ABIs to torch tensors share: reading arguments, the current
// stream, errors, and the entries of a CPython module without the dispatcher in front. A binding defines
// BINDING_TAG, the words before its errors, BINDING_ERROR, its library's last error, and includes this
// first. Everything here is local to the file that includes it.
#pragma once
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <stdexcept>
#include <string>

namespace {

using at::Tensor;

[[noreturn]] void fail(const char* op, const std::string& what) {
  throw std::runtime_error(std::string(BINDING_TAG) + op + ": " + what);
}

std::string str(long x) { return std::to_string(x); }
std::string str(const Tensor& t) {
  if (!t.defined()) return "None";
  std::string s = std::string(c10::toString(t.scalar_type())) + " [";
  for (long i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + str(t.size(i));
  return s + "]";
}

// ---- arguments ----------------------------------------------------------------------------------
struct Args {
  const char* op;
  PyObject* const* at;

  Tensor tensor(int i) const {
    if (!THPVariable_Check(at[i])) fail(op, "argument " + str(i) + " must be a tensor");
    return THPVariable_Unpack(at[i]);
  }
  Tensor optional(int i) const { return at[i] == Py_None ? Tensor() : tensor(i); }
  bool flag(int i) const { return PyObject_IsTrue(at[i]) == 1; }
  double real(int i) const {
    const double x = PyFloat_AsDouble(at[i]);
    if (PyErr_Occurred()) throw python_error();
    return x;
  }
  int integer(int i, const char* name) const {
    const long x = PyLong_AsLong(at[i]);
    if (PyErr_Occurred()) throw python_error();
    return to_int(x, name);
  }
  int to_int(long x, const char* name) const {
    if (x > INT_MAX || x < INT_MIN) fail(op, std::string(name) + "=" + str(x) + " is out of range");
    return (int)x;
  }
};

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
template <typename T>
T* address_as(const Tensor& t) { return t.defined() ? (T*)const_cast<void*>(t.const_data_ptr()) : nullptr; }

c10::Device device_of(const char* op, std::initializer_list<const Tensor*> tensors) {
  const c10::Device dev = (*tensors.begin())->device();
  if (!dev.is_cuda()) fail(op, "tensors must be on the GPU, got " + dev.str());
  for (const Tensor* t : tensors)
    if (t->defined() && t->device() != dev) fail(op, "tensors on " + dev.str() + " and " + t->device().str());
  return dev;
}

void check(int status) {
  if (status) throw std::runtime_error(std::string(BINDING_TAG) + BINDING_ERROR());
}

// A launch, with the interpreter free meanwhile: it waits where the stream's queue is full.
template <typename F>
void launch(c10::Device dev, F f) {
  void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  PyThreadState* state = PyEval_SaveThread();
  const int status = f(stream);
  PyEval_RestoreThread(state);
  check(status);
}

// A tensor that a launch has written: what autograd saved of it before is out of date.
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor new_bf16(c10::Device dev, at::IntArrayRef shape) {
  return at::empty(shape, at::TensorOptions().dtype(at::kBFloat16).device(dev));
}

Tensor ints(const Args& a, const char* name, const Tensor& t, at::ScalarType type, long n,
            const char* what) {
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n)
    fail(a.op, std::string(name) + " must be " + what + " [" + str(n) + "], got " + str(t));
  return t.contiguous();
}

// What the dispatcher resolves before an op sees it: the tensors of transforms (vmap's have no storage),
// subclasses with a dispatch of their own, views that stand for other values than their bytes.
constexpr c10::DispatchKeySet kNotPlain({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                         c10::DispatchKey::Functionalize, c10::DispatchKey::Python,
                                         c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                         c10::DispatchKey::ZeroTensor});

// Whether the tensors among the arguments may be taken as they are, past the dispatcher: none is of a
// subclass or of those keys, and no gradient is asked of any.
bool plain(PyObject* const* args, Py_ssize_t n) {
  const bool grad = c10::GradMode::is_enabled();
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* x = args[i];
    if (x == Py_None || PyLong_Check(x) || PyFloat_Check(x)) continue;
    if (!THPVariable_CheckExact(x)) {     // (a Parameter is exact)
      if (THPVariable_Check(x)) return false;
      continue;
    }
    const Tensor& t = THPVariable_Unpack(x);
    if (t.key_set().has_any(kNotPlain) || (grad && t.requires_grad())) return false;
  }
  return true;
}

// Nothing thrown leaves an entry: torch's handlers turn it into the Python exception.
template <PyObject* (*F)(const Args&), int N, bool IfPlain>
PyObject* entry(const char* op, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) fail(op, str(n) + " arguments in place of " + str(N));
  if (IfPlain && !plain(args, n)) Py_RETURN_NOTIMPLEMENTED;
  return F(Args{op, args});
  END_HANDLE_TH_ERRORS
}
PyObject* is_plain(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return PyBool_FromLong(plain(args, n));
  END_HANDLE_TH_ERRORS
}
#define METHOD(name, f) {name, (PyCFunction)(void (*)(void))(_PyCFunctionFast)f, METH_FASTCALL, nullptr}
#define ENTRY(name, n, if_plain)                                                                 \
  [](PyObject*, PyObject* const* a, Py_ssize_t k) -> PyObject* {                                 \
    return entry<name, n, if_plain>(#name, a, k);                                                \
  }
// name, and name_if_plain, which returns NotImplemented where the tensors are not
#define ENTRIES(name, n) METHOD(#name, ENTRY(name, n, false)), METHOD(#name "_if_plain", ENTRY(name, n, true))

}  // namespace
