// What the native layers share: Python's exceptions from code that runs with or without the interpreter lock, argument checks, the current stream
// and the count of launches.
#pragma once
#include <torch/extension.h>

#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <atomic>
#include <string>

#include "b200ops.h"

namespace b200torch {

namespace py = pybind11;
using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// Of this copy of the module alone, should a process load two.
extern __attribute__((visibility("hidden"))) std::atomic<int64_t> g_launches;
extern __attribute__((visibility("hidden"))) PyObject* g_error;   // the package's B200OpsError (a RuntimeError), looked up when the module is loaded

// Raises a Python exception with or without the interpreter lock: with it as error_already_set, without (in a
// layer's body, forward or on an autograd thread) in torch's own carrier.
[[noreturn]] inline void raise(PyObject* type, const std::string& what) {
  if (PyGILState_Check()) {
    PyErr_SetString(type, what.c_str());
    throw py::error_already_set();
  }
  py::gil_scoped_acquire gil;
  PyErr_SetString(type, what.c_str());
  python_error err;
  err.persist();
  throw err;
}
inline void require(bool ok, const char* what) {
  if (!ok) raise(PyExc_AssertionError, what);
}
// Rows of `width` elements; an empty row is the error that the division is in Python, not a signal.
inline int64_t rows_of(const Tensor& t, int64_t width) {
  if (width == 0) raise(PyExc_ZeroDivisionError, "the last dimension holds no element of a row");
  return t.numel() / width;
}
inline void check(int rc, const char* what) {
  if (rc != 0) raise(g_error, std::string(what) + " failed with code " + std::to_string(rc));
}
inline bool bf16_cuda(const Tensor& t) { return t.is_cuda() && t.scalar_type() == at::kBFloat16; }
// An incoming gradient as the kernels read it: contiguous and on a 16-byte boundary, whatever view it is.
inline Tensor rows16(const Tensor& g) {
  const Tensor c = g.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
inline void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// pybind's exception cannot cross the autograd engine's threads; torch's carrier can.
template <class F>
auto on_engine_thread(F f) {
  try {
    return f();
  } catch (py::error_already_set& e) {
    py::gil_scoped_acquire gil;
    e.restore();
    python_error err;
    err.persist();
    throw err;
  }
}

// The call itself, or under torch.jit.trace the operator of the same name: the tracer records operators,
// and of the bodies above it would see nothing but the allocation of their outputs.
template <class R, class... A, class... Args>
R traced_or_direct(const char* name, R (*fn)(A...), const Args&... args) {
  if (!torch::jit::tracer::isTracing()) return fn(args...);
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<R(A...)>().call(args...);
}

// The layers of a mixture-of-experts block and its optimizer's step (torch_moe.cpp)
void bind_moe(py::module_& m);

}  // namespace b200torch
