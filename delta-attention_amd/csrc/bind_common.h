// What the extension modules of the Python calls share: checks of arguments,
// tensors as the kernels take them, the current stream, errors. Included by one
// source file of each module.
//
// Problems with the arguments are AssertionErrors, as the other calls'.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <limits>
#include <stdexcept>
#include <string>

#include "delta_attn.h"

namespace {

PyObject* g_check;         // _lib.check, handed over by the module's bind()

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct PythonError {};     // a Python exception is set

#define REQUIRE(cond, ...) \
  if (!(cond)) throw Refused(c10::str(__VA_ARGS__))

PyObject* new_ref(PyObject* o) {
  Py_INCREF(o);
  return o;
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  REQUIRE(THPVariable_Check(o), what, ": a tensor is needed");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (!i) throw PythonError();
  const long long x = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (x == -1 && PyErr_Occurred()) throw PythonError();
  return x;
}

int32_t narrow(int64_t x, const char* what) {
  REQUIRE(x >= 0 && x <= std::numeric_limits<int32_t>::max(), what, ": ", x, " is out of range");
  return (int32_t)x;
}

int32_t dtype_code(at::ScalarType t) {
  REQUIRE(t == at::kBFloat16 || t == at::kHalf, "dtype ", t, " is not supported (bfloat16, float16)");
  return t == at::kBFloat16 ? DA_BF16 : DA_FP16;
}

void on_gpu(c10::Device dev) { REQUIRE(dev.is_cuda(), "delta-attention kernels need GPU tensors"); }

// Rows contiguous and 16-byte aligned, as the kernels read them (a copy where
// they are not); the strides of dimensions of one entry do not count.
at::Tensor ready(const at::Tensor& t) {
  int64_t bits = 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) bits |= t.size(i) > 1 ? t.stride(i) : 0;
  const bool ok = t.stride(-1) == 1 && !(bits & 7) && (uintptr_t)t.data_ptr() % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// (entries of one-entry dimensions are never stepped over)
void strides3(int64_t* to, const at::Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// An optional device tensor of one entry, or one per sequence -> its pointer;
// `per_seq` whether the latter.
template <typename T>
const T* entries(PyObject* o, int64_t B, at::ScalarType type, c10::Device dev, const char* what, int32_t& per_seq) {
  per_seq = 0;
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, what);
  REQUIRE(t.scalar_type() == type && t.device() == dev && t.dim() <= 1 && (t.numel() == 1 || t.numel() == B) && t.is_contiguous(),
          what, ": a contiguous ", type, " tensor of 1 or ", B, " entries on ", dev, " is needed, got ", t.scalar_type(),
          t.sizes(), " on ", t.device());
  per_seq = t.numel() == B;
  return (const T*)t.data_ptr();
}

// The device of the call's tensors as the current one; its current stream.
class On {
 public:
  explicit On(c10::Device dev) {
    if (hipGetDevice(&before_) != hipSuccess) throw std::runtime_error("no current GPU");
    now_ = dev.index();
    if (now_ != before_ && hipSetDevice(now_) != hipSuccess) throw std::runtime_error("cannot switch to the tensors' GPU");
  }
  ~On() {
    if (now_ != before_) (void)hipSetDevice(before_);
  }
  void* stream() const { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)now_).stream(); }

 private:
  int before_ = 0, now_ = 0;
};

void check(int rc, const char* what) {
  if (rc == DA_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, what);
  Py_XDECREF(r);
  if (PyErr_Occurred()) throw PythonError();
  throw std::runtime_error(std::string(what) + " failed");
}

PyObject* bind(PyObject* const* a);     // each module's own: the library's functions

// Argument count and exceptions, at the border to Python.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%zd arguments are needed, got %zd", N, n);
    return nullptr;
  }
  try {
    if (F != &bind && !g_check) throw std::runtime_error("the library is not bound");
    return F(args);
  } catch (const PythonError&) {
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_AssertionError, e.what());
  } catch (...) {            // torch's own errors keep their types (out of memory)
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

}  // namespace
