// What the Python bindings share: tensors' checks, the device and stream of a call,
// errors as Python exceptions.
//
// Errors: ValueError for malformed arguments, NotImplementedError for what the
// kernels do not take, RuntimeError for tensors in the wrong place and CUDA
// failures, TypeError for what is no tensor.  No C++ exception leaves a function.
#pragma once

#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <string>
#include <utility>

#include "logitfill_b200.h"

namespace {

struct Fail {
  PyObject* type;
  std::string text;
};
template <typename... A>
[[noreturn]] void fail(PyObject* type, const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Fail{type, s.str()};
}

std::string shape(const at::Tensor& t) {
  std::ostringstream s;
  s << c10::toString(t.scalar_type()) << " [";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << "] on " << t.device();
  return s.str();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

// For operators that record no gradient, of either direction: a result that silently dropped
// it would be wrong.
[[maybe_unused]] void no_gradient(const at::Tensor& t, const char* what) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    fail(PyExc_NotImplementedError, what, " requires a gradient, which this operator does not record: call it under torch.no_grad()");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    fail(PyExc_NotImplementedError, what, " has a forward-mode tangent, which this operator does not carry on");
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LF_F32;
    case at::kHalf: return LF_F16;
    case at::kBFloat16: return LF_BF16;
    default:
      fail(PyExc_NotImplementedError, "dtype ", c10::toString(t), " is not supported (float32, float16, bfloat16)");
  }
}

// t [B, H, T, D] with 16-byte aligned rows of channel stride 1 (a copy where it is
// not), and its first three strides (0 where the extent is 1).
at::Tensor aligned_rows(at::Tensor t, int64_t (&s)[3]) {
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    const auto address = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.stride(3) == 1 && address % 16 == 0 && (s[0] | s[1] | s[2]) * static_cast<int64_t>(t.element_size()) % 16 == 0) break;
    t = t.clone(at::MemoryFormat::Contiguous);
  }
  return t;
}

// Whether two tensors are known to share memory (strided views of one buffer whose gaps
// hold the other are not: q and k of one projection).
bool overlap(const at::Tensor& x, const at::Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  const at::MemOverlapStatus s = at::get_overlap_status(x, y);
  return s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial;
}

// The device a call runs on made current, and its stream.
struct Launch {
  c10::cuda::OptionalCUDAGuard guard;
  c10::cuda::CUDAStream stream;
  explicit Launch(at::Device d) : guard(d), stream(c10::cuda::getCurrentCUDAStream(d.index())) {}
  lf_stream_t raw() const { return reinterpret_cast<lf_stream_t>(stream.stream()); }
};

void check(int status, const char* what) {
  if (status == LF_OK) return;
  fail(status == LF_ERR_UNSUPPORTED        ? PyExc_NotImplementedError
       : status == LF_ERR_INVALID_ARGUMENT ? PyExc_ValueError
                                           : PyExc_RuntimeError,
       what, ": ", lf_status_string(status), ": ", lf_last_error());
}

template <typename F>
PyObject* guarded(F&& body) noexcept {
  try {
    return body();
  } catch (const Fail& f) {
    PyErr_SetString(f.type, f.text.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

void expect(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) fail(PyExc_TypeError, "expected ", want, " arguments, got ", got);
}
int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    fail(PyExc_TypeError, name, " must be an integer");
  }
  return v;
}

bool truth(PyObject* o, const char* name) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    fail(PyExc_TypeError, name, " must be true or false");
  }
  return v != 0;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

}  // namespace
