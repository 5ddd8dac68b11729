// What the native host path's translation units share: errors, streams, and the conditions under which a call is made as a node of its own.
#pragma once
#include <torch/extension.h>
#include <ATen/SavedTensorHooks.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/Exceptions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/spion_b200.h"

namespace spion_torch {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using c10::optional;

struct Failure : std::runtime_error { using std::runtime_error::runtime_error; };

inline void check(int rc, const char* what) {
  if (rc != 0) throw Failure(std::string(what) + " failed: " + spion_status_string(rc) + " (" + std::to_string(rc) + ")");
}

inline py::object& error_type() {
  static py::object* type = new py::object(py::module_::import("spion_b200._lib").attr("SpionError"));      // never destroyed
  return *type;
}
// A backward runs on a thread of the autograd engine, which turns C++ exceptions into RuntimeError: raise the library's own
// error there, as the forward does through the module's exception translator.
template <class F>
variable_list as_backward(F f) {
  try {
    return f();
  } catch (const Failure& e) {
    py::gil_scoped_acquire gil;
    PyErr_SetString(error_type().ptr(), e.what());
    python_error raised;
    raised.persist();
    throw raised;
  }
}

inline void* stream_of(const Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
inline void* p(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline const float* pf(const Tensor& t) { return t.defined() ? (const float*)t.data_ptr() : nullptr; }

// The nodes below work on memory: they form no forward-mode tangents, and tracers, dispatch modes and transforms would not see what
// they do.  Calls under one of those take the way over torch operators and Python autograd functions, which they know.
inline bool plain(const Tensor& t) {
  static const c10::DispatchKeySet wrapped({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::FuncTorchGradWrapper,
                                            c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Functionalize, c10::DispatchKey::Negative,
                                            c10::DispatchKey::ZeroTensor});
  return !t.key_set().has_any(wrapped) && !t._fw_grad(0).defined();
}
inline bool plain(std::initializer_list<at::ArrayRef<Tensor>> lists) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
  for (const auto& ts : lists)
    for (const Tensor& t : ts)
      if (!plain(t)) return false;
  return true;
}

inline SavedVariable save(const Tensor& t) { return SavedVariable(t, false); }

// A backward that is itself recorded (create_graph)
inline bool recorded() { return at::GradMode::is_enabled(); }
struct OutsideAutocast { c10::impl::ExcludeDispatchKeyGuard guard{c10::autocast_dispatch_keyset}; };

// torch_encoder_ops.cpp
void add_encoder_ops(py::module_& m);

}  // namespace spion_torch

using namespace spion_torch;
