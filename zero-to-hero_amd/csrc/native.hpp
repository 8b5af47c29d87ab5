// Shared pieces of ppo_amd._native's sources: argument checks, streams, results
// and the entry points' frame.
#pragma once

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/SavedTensorHooks.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Generator.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "ppo_amd.h"

namespace ppo_native {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// What init() hands over: the workspace pool, the LossStats class, the function
// that raises for a library error code, and torch.nn's classes.
struct Python {
  PyObject* pool = nullptr;
  PyObject* stats = nullptr;
  PyObject* fail = nullptr;
  PyObject *sequential = nullptr, *linear = nullptr, *relu = nullptr, *tanh = nullptr;
  PyObject* scalar_names[PPO_NUM_SCALARS] = {};
  PyObject *get = nullptr, *modules = nullptr, *parameters = nullptr, *net = nullptr,
           *weight = nullptr, *bias = nullptr, *in_features = nullptr, *out_features = nullptr;
};
extern Python P;

// Thrown for a call that is not the ordinary one (entry clears a Python error that
// a look at its arguments has set).
struct NotPlain {};

inline void need(bool ok) {
  if (!ok) throw NotPlain{};
}

// Modes, transforms and traces that want to see torch operators or autograd
// functions: not for this path.
inline bool plain_mode() {
  return !torch::jit::tracer::isTracing() && !at::impl::torch_function_mode_enabled() &&
         !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !c10::impl::tls_is_dispatch_key_included(
             c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

inline void need_plain_mode() { need(plain_mode()); }

// Keys of tensors that stand for another tensor, or for none: no storage of
// their own to read.
constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::Python, c10::DispatchKey::Batched,
                                        c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper,
                                        c10::DispatchKey::Functionalize,
                                        c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                        c10::DispatchKey::ZeroTensor});

// A torch.Tensor (or Parameter) itself: no subclass, no wrapper, dense GPU
// storage, contiguous.
inline const Tensor& plain(PyObject* o, at::ScalarType type) {
  need(THPVariable_CheckExact(o));
  const Tensor& t = THPVariable_Unpack(o);
  need(t.defined() && t.is_cuda() && t.layout() == at::kStrided &&
       !t.key_set().has_any(kWrapped) && t.scalar_type() == type && t.is_contiguous());
  return t;
}

inline const Tensor& plain(PyObject* o, at::ScalarType type, const at::Device& device) {
  const Tensor& t = plain(o, type);
  need(t.device() == device);
  return t;
}

inline const Tensor& plain_rows(PyObject* o, const at::Device& device, int64_t n) {
  const Tensor& t = plain(o, at::kFloat, device);
  need(t.dim() == 1 && t.size(0) == n);
  return t;
}

inline double number(PyObject* o) {
  need(PyFloat_CheckExact(o) || PyLong_CheckExact(o));
  const double x = PyFloat_AsDouble(o);
  need(x != -1.0 || !PyErr_Occurred());
  return x;
}

inline int64_t integer(PyObject* o) {
  const int64_t x = PyLong_AsLongLong(o);
  need(x != -1 || !PyErr_Occurred());
  return x;
}

inline const float* in(const Tensor& t) { return t.const_data_ptr<float>(); }
inline float* out(const Tensor& t) { return t.data_ptr<float>(); }

inline void* current_stream(const at::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

// Allocations and the library call, outside the GIL: other Python threads run
// while this one waits for memory or for room in a full hardware queue.
template <typename F>
int unlocked(F f) {
  py::gil_scoped_release no_gil;
  return f();
}

// Raises PPOLibraryError (ops._native_failed) for a non-zero status.
inline void check(const char* name, int code, const at::Device& device, void* stream) {
  if (code == PPO_OK) return;
  py::object dev = py::reinterpret_steal<py::object>(THPDevice_New(device));
  py::reinterpret_borrow<py::object>(P.fail)(name, code, dev,
                                             reinterpret_cast<uintptr_t>(stream));
}

// The same inside an autograd node, where the GIL may be held by nobody.
inline void check_in_node(const char* name, int code, const at::Device& device, void* stream) {
  if (code == PPO_OK) return;
  py::gil_scoped_acquire gil;
  try {
    check(name, code, device, stream);
  } catch (py::error_already_set& e) {
    e.restore();
    python_error error;
    error.persist();
    throw std::move(error);
  }
}

inline PyObject* wrap(const Tensor& t) {
  PyObject* o = THPVariable_Wrap(t);
  if (!o) throw py::error_already_set();
  return o;
}

inline PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  py::tuple r(ts.size());
  size_t k = 0;
  for (const Tensor& t : ts) PyTuple_SET_ITEM(r.ptr(), k++, wrap(t));
  return r.release().ptr();
}

template <PyObject* (*kFn)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != kArgs) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    need(P.pool != nullptr);
    need_plain_mode();
    return kFn(args);
  } catch (const NotPlain&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  } catch (py::error_already_set& e) {
    e.restore();
    return nullptr;
  } catch (python_error& e) {
    e.restore();
    return nullptr;
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

#define PPO_ENTRY(name, fn, nargs) \
  {name, (PyCFunction)(void (*)(void))(&entry<fn, nargs>), METH_FASTCALL, nullptr}

}  // namespace ppo_native
