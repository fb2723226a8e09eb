// What the Python bindings of the C ABI share: arguments taken from Python objects, checks, and
// exceptions translated.  Everything has internal linkage: each binding is a module of its own.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <stdexcept>
#include <string>

#include "vggt_sparse.h"

namespace {

struct ValueError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

[[noreturn]] void refuse(const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  throw ValueError(text);
}

// A tensor argument, or none.
const at::Tensor* tensor_or_none(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o, const char* name) {
  const at::Tensor* t = tensor_or_none(o, name);
  if (!t) refuse("%s must be a tensor", name);
  return *t;
}

double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse("%s must be a number", name);
  }
  return v;
}
int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse("%s must be an integer", name);
  }
  return v;
}
bool truth(PyObject* o, const char* name) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    refuse("%s must be a truth value", name);
  }
  return v == 1;
}

void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// The status word (int32), or none.
int32_t* status_of(const at::Tensor* t) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kInt || t->numel() < 1)
    refuse("status must be an int32 tensor with at least one element");
  return static_cast<int32_t*>(t->data_ptr());
}

// All on one CUDA device (there is no CPU path).
template <typename... Ts>
c10::Device one_device(const at::Tensor& first, const Ts*... rest) {
  const c10::Device d = first.device();
  bool cuda = d.is_cuda(), same = true;
  ((cuda = cuda && (!rest || rest->is_cuda()), same = same && (!rest || rest->device() == d)), ...);
  if (!cuda) refuse("vggt_sparse operators take CUDA tensors (there is no CPU path)");
  if (!same) refuse("the tensors must be on one device");
  return d;
}

void check(int rc) {
  if (rc == 0) return;
  const char* text = vggt_sparse_last_error();
  if (rc < 0) throw ValueError(text);
  throw std::runtime_error(text);
}

template <typename F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F&& body) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, have);
    return nullptr;
  }
  try {
    return body();
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyObject* returned(PyObject* given, const at::Tensor& t) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(t);
}

}  // namespace
