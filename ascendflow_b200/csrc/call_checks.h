// What the native host side's checks and calls share: arguments from Python, what a tensor has to be, results, the registered ops' way to the front end.
#pragma once

#include "host_calls.h"

#include <ATen/core/grad_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <functional>
#include <optional>
#include <vector>

#include "../../include/latent.h"

namespace ascendflow_host {

using Tensor = at::Tensor;

// A plain torch.Tensor argument, or nullptr.
inline const Tensor* tensor_of(PyObject* object) { return THPVariable_CheckExact(object) ? &THPVariable_Unpack(object) : nullptr; }

// The same for an argument that may be None (*present tells); false for anything else.
inline bool optional_of(PyObject* object, const Tensor** tensor) {
  *tensor = object == Py_None ? nullptr : tensor_of(object);
  return object == Py_None || *tensor != nullptr;
}

inline bool on_device(const Tensor& t, int device, at::ScalarType type) {
  return t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.device().index() == device && t.scalar_type() == type &&
         !t.is_conj() && !t.is_neg() && !(t.requires_grad() && at::GradMode::is_enabled()) && !t._fw_grad(0).defined();
}
inline bool shaped(const Tensor& t, std::initializer_list<int64_t> sizes) {
  return t.dim() == int64_t(sizes.size()) && std::equal(sizes.begin(), sizes.end(), t.sizes().begin());
}
inline bool plain(const Tensor& t, int device, at::ScalarType type, std::initializer_list<int64_t> sizes) {
  return on_device(t, device, type) && t.is_contiguous() && shaped(t, sizes);
}
// The stride of a dimension; that of one with at most one entry counts for nothing.
inline int64_t stride_of(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }
// Entries of the last dimension follow each other; rows start on 16-byte boundaries.
inline bool rows_aligned(const Tensor& t) {
  const int64_t last = t.dim() - 1, size = t.element_size();
  if (t.numel() == 0) return true;
  if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0 || (t.size(last) > 1 && t.stride(last) != 1)) return false;
  for (int64_t d = 0; d < last; ++d)
    if (stride_of(t, d) * size % 16 != 0) return false;
  return true;
}
// No two entries share memory.
inline bool entries_apart(const Tensor& t) {
  std::array<std::pair<int64_t, int64_t>, 4> dims;
  int64_t extent = 1;
  const int count = int(t.dim());
  for (int d = 0; d < count; ++d) dims[d] = {t.size(d) > 1 ? t.stride(d) : 0, t.size(d)};
  std::sort(dims.begin(), dims.begin() + count);
  for (int d = 0; d < count; ++d) {
    if (dims[d].second <= 1) continue;
    if (dims[d].first < extent) return false;
    extent += dims[d].first * (dims[d].second - 1);
  }
  return true;
}
inline std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  if (t.numel() == 0) return {begin, begin};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += t.stride(d) * (t.size(d) - 1);
  return {begin, begin + uintptr_t(last + 1) * t.element_size()};
}
inline bool disjoint(const Tensor& a, const Tensor& b) {
  const auto x = span(a), y = span(b);
  return x.first == x.second || y.first == y.second || x.second <= y.first || y.second <= x.first;
}

inline PyObject* real_numbers = nullptr;  // numbers.Real

// A real number of any kind, but no tensor: that would have to be waited for.
inline bool number_of(PyObject* object, double* value) {
  if (!PyFloat_Check(object) && !PyLong_Check(object)) {
    const int real = real_numbers == nullptr ? 0 : PyObject_IsInstance(object, real_numbers);
    if (real < 0) PyErr_Clear();
    if (real != 1) return false;
  }
  *value = PyFloat_AsDouble(object);
  if (*value == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
inline bool flag_of(PyObject* object, bool* value) {
  if (!PyBool_Check(object)) return false;
  *value = object == Py_True;
  return true;
}

inline int32_t type_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? LATENT_BF16 : t.scalar_type() == at::kHalf ? LATENT_F16 : t.scalar_type() == at::kFloat ? LATENT_F32 : -1;
}
inline void* memory(const Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }
template <typename T> T* memory_as(const Tensor& t) { return static_cast<T*>(memory(t)); }

// A tensor allocated on another stream: its memory must not be recycled before this one is done with it.
inline void used_on(const c10::cuda::CUDAStream& stream, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t != nullptr) c10::cuda::CUDACachingAllocator::recordStream(t->storage().data_ptr(), stream);
}

inline PyObject* raise_launch_status(int status) {
  PyErr_Format(PyExc_RuntimeError, "kernel launch failed with status %d; device retries are disabled", status);
  return nullptr;
}
// What was written in place counts its version up, as for any in-place operation (a tensor made in inference mode has none).
inline void count_up(const Tensor* t) {
  if (t != nullptr && t->defined() && !t->is_inference()) torch::autograd::increment_version(*t);
}

// Each call: checks and launch. kRefused: not accepted, nothing enqueued; otherwise the launch's status.
constexpr int kRefused = -1000;

// True, False for a refused call, or an error.
inline PyObject* finished(int status, std::initializer_list<const Tensor*> written) {
  if (status == kRefused) Py_RETURN_FALSE;
  if (status != 0) return raise_launch_status(status);
  for (const Tensor* t : written) count_up(t);
  Py_RETURN_TRUE;
}

// Plain tensors in the first arguments, and nobody who wants to see what is called (a dispatch mode, as in tracing; the front end then calls the registered op).
template <size_t N>
inline bool tensors_of(PyObject* const* arguments, std::array<const Tensor*, N>* tensors) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
  for (size_t i = 0; i < N; ++i)
    if (((*tensors)[i] = tensor_of(arguments[i])) == nullptr) return false;
  return true;
}

inline PyObject* checked_call = nullptr;  // the front end's call, for arguments refused here

// What the launch said; a refused call goes through the front end, (name, arguments ...), which words the error.
inline void settle(int status, const char* name, std::initializer_list<std::function<PyObject*()>> arguments) {
  if (status == 0) return;
  pybind11::gil_scoped_acquire gil;
  PyObject* result = nullptr;
  if (status == kRefused && checked_call != nullptr) {
    PyObject* call = PyTuple_New(Py_ssize_t(arguments.size()) + 1);
    Py_ssize_t at = 0;
    PyTuple_SET_ITEM(call, at++, PyUnicode_FromString(name));
    for (const auto& argument : arguments) PyTuple_SET_ITEM(call, at++, argument());
    result = PyObject_CallObject(checked_call, call);
    Py_DECREF(call);
  } else {
    raise_launch_status(status);
  }
  if (result == nullptr) {
    python_error error;
    error.persist();
    throw error;
  }
  Py_DECREF(result);
}
inline auto boxed(const Tensor& t) {
  return [&t] { return THPVariable_Wrap(t); };
}
inline auto boxed(const std::optional<Tensor>& t) {
  return [&t] { return t.has_value() ? THPVariable_Wrap(*t) : Py_NewRef(Py_None); };
}
inline auto boxed(double value) {
  return [value] { return PyFloat_FromDouble(value); };
}
inline auto boxed(int64_t value) {
  return [value] { return PyLong_FromLongLong(value); };
}
inline auto boxed(at::TensorList tensors) {
  return [tensors] {
    PyObject* list = PyList_New(Py_ssize_t(tensors.size()));
    for (size_t i = 0; i < tensors.size(); ++i) PyList_SET_ITEM(list, Py_ssize_t(i), THPVariable_Wrap(tensors[i]));
    return list;
  };
}
inline auto boxed(bool value) {
  return [value] { return PyBool_FromLong(value); };
}
inline std::vector<Tensor> tensors_in(const c10::IValue& argument) {
  if (argument.isTensor()) return {argument.toTensor()};
  return argument.isTensorList() ? argument.toTensorVector() : std::vector<Tensor>{};
}

// No gradient: tensors that want one are refused, also while a graph is traced.
inline void without_gradient(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  if (at::GradMode::is_enabled())
    for (const c10::IValue& argument : torch::jit::last(*stack, op.schema().arguments().size()))
      for (const Tensor& t : tensors_in(argument)) TORCH_CHECK(!t.defined() || !t.requires_grad(), op.schema().name(), ": the operator has no gradient");
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

// What is written in place counts its version up.
inline void mutates(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const auto& parameters = op.schema().arguments();
  const auto arguments = torch::jit::last(*stack, parameters.size());
  std::vector<Tensor> written;
  for (size_t i = 0; i < parameters.size(); ++i)
    if (parameters[i].alias_info() != nullptr && parameters[i].alias_info()->isWrite())
      for (const Tensor& t : tensors_in(arguments[i])) written.push_back(t);
  {
    at::AutoDispatchBelowADInplaceOrView below;
    op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
  }
  for (const Tensor& t : written) count_up(&t);
}

template <PyObject* (*function)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)); }


}  // namespace ascendflow_host
