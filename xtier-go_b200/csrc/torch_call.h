// What the Python package's bindings share: torch tensors and integers taken from a call's arguments, refusals that become
// the package's error class, the current stream of the tensors' device. XTG_NAME (a string) starts every message.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../../include/xtg_cuda.h"

namespace {

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

PyObject* error_class = nullptr;

void require(bool ok, const std::string& why) {
  if (!ok) throw Refused(XTG_NAME ": " + why);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  require(THPVariable_Check(o), std::string(name) + " is a tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused(std::string(XTG_NAME ": ") + name + " is an integer");
  }
  return v;
}

int small(PyObject* o, const char* name) {
  const int64_t v = integer(o, name);
  require(v >= INT32_MIN && v <= INT32_MAX, std::string(name) + " is a 32-bit integer");
  return (int)v;
}

int code_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

void require_index(const char* name, const at::Tensor& t, int dims, c10::Device dev) {
  require(t.scalar_type() == at::kInt && t.dim() == dims && t.device() == dev && t.is_contiguous(),
          std::string(name) + " is a contiguous int32 tensor of " + std::to_string(dims) +
              " dimension(s) on the pool's device");
}

// The stride of dimension d; that of a single row or head, which nothing steps by, may be any number.
int64_t stride(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Runs f (which gets the current stream and a message buffer) with device dev current.
template <class F>
void call(c10::Device dev, F&& f) {
  char why[1024] = "";
  const c10::cuda::CUDAGuard guard(dev);
  if (f(c10::cuda::getCurrentCUDAStream(dev.index()).stream(), why, (int)sizeof(why)) != 0) throw Refused(why);
}

// A METH_FASTCALL function of n arguments; C++ exceptions end here, as the package's error class.
template <class F>
PyObject* entry(const char* name, Py_ssize_t given, Py_ssize_t wanted, F&& f) {
  try {
    require(error_class != nullptr, "bind first");
    require(given == wanted, std::string(name) + " takes " + std::to_string(wanted) + " arguments");
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, XTG_NAME ": unknown error");
  }
  return nullptr;
}

}  // namespace
