// The host side of the operators around dense latent attention: checks and launches, as host_calls.cpp does them for
// the sparse operator. A call that passes is launched through the C ABI and the function returns True; for one that does
// not it returns False without having enqueued anything, and `latent.py` finds the violated rule and words the error.

#include "host_calls.h"

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <limits>

#include "../../include/latent.h"

namespace {

using Tensor = at::Tensor;

decltype(&launch_latent_rotary) launch_rotary = nullptr;
decltype(&launch_latent_append) launch_append = nullptr;
decltype(&launch_latent_attention) launch_attention = nullptr;
decltype(&launch_latent_prefill) launch_prefill = nullptr;
decltype(&workspace_size_latent_attention) workspace_size = nullptr;
decltype(&workspace_size_latent_prefill) prefill_workspace_size = nullptr;

constexpr double kLeastScale = 1e-30, kMostScale = 1e30;  // what FP32 holds with room to spare
constexpr int64_t kMostRows = int64_t(1) << 30;  // tokens x heads

// A plain torch.Tensor argument, or nullptr.
const Tensor* tensor_of(PyObject* object) { return THPVariable_CheckExact(object) ? &THPVariable_Unpack(object) : nullptr; }

// The same for an argument that may be None (*present tells); false for anything else.
bool optional_of(PyObject* object, const Tensor** tensor) {
  *tensor = object == Py_None ? nullptr : tensor_of(object);
  return object == Py_None || *tensor != nullptr;
}

bool on_device(const Tensor& t, int device, at::ScalarType type) {
  return t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.device().index() == device && t.scalar_type() == type &&
         !t.is_conj() && !t.is_neg() && !(t.requires_grad() && at::GradMode::is_enabled()) && !t._fw_grad(0).defined();
}
bool shaped(const Tensor& t, std::initializer_list<int64_t> sizes) {
  return t.dim() == int64_t(sizes.size()) && std::equal(sizes.begin(), sizes.end(), t.sizes().begin());
}
bool plain(const Tensor& t, int device, at::ScalarType type, std::initializer_list<int64_t> sizes) {
  return on_device(t, device, type) && t.is_contiguous() && shaped(t, sizes);
}
// The stride of a dimension; that of one with at most one entry counts for nothing.
int64_t stride_of(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }
// Entries of the last dimension follow each other; rows start on 16-byte boundaries.
bool rows_aligned(const Tensor& t) {
  const int64_t last = t.dim() - 1, size = t.element_size();
  if (t.numel() == 0) return true;
  if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0 || (t.size(last) > 1 && t.stride(last) != 1)) return false;
  for (int64_t d = 0; d < last; ++d)
    if (stride_of(t, d) * size % 16 != 0) return false;
  return true;
}
// No two entries share memory.
bool entries_apart(const Tensor& t) {
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
std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  if (t.numel() == 0) return {begin, begin};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += t.stride(d) * (t.size(d) - 1);
  return {begin, begin + uintptr_t(last + 1) * t.element_size()};
}
bool disjoint(const Tensor& a, const Tensor& b) {
  const auto x = span(a), y = span(b);
  return x.first == x.second || y.first == y.second || x.second <= y.first || y.second <= x.first;
}

PyObject* real_numbers = nullptr;  // numbers.Real

// A real number of any kind, but no tensor: that would have to be waited for.
bool number_of(PyObject* object, double* value) {
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
  return std::isfinite(*value);
}
// What cosines and sines are multiplied by, in FP32.
bool amplitude_of(PyObject* object, double* value) { return number_of(object, value) && std::abs(*value) <= std::numeric_limits<float>::max(); }
bool flag_of(PyObject* object, int32_t* value) {
  if (!PyBool_Check(object)) return false;
  *value = object == Py_True;
  return true;
}

int32_t type_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? LATENT_BF16 : t.scalar_type() == at::kHalf ? LATENT_F16 : t.scalar_type() == at::kFloat ? LATENT_F32 : -1;
}
void* memory(const Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }
template <typename T> T* memory_as(const Tensor& t) { return static_cast<T*>(memory(t)); }

// A tensor allocated on another stream: its memory must not be recycled before this one is done with it.
void used_on(const c10::cuda::CUDAStream& stream, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t != nullptr) c10::cuda::CUDACachingAllocator::recordStream(t->storage().data_ptr(), stream);
}

// Behind the launch. What was written in place counts its version up, as for any in-place operation (a tensor made in inference mode has none).
PyObject* finished(int status, std::initializer_list<const Tensor*> written) {
  if (status == 0) {
    for (const Tensor* t : written)
      if (t != nullptr && !t->is_inference()) torch::autograd::increment_version(*t);
    Py_RETURN_TRUE;
  }
  PyErr_Format(PyExc_RuntimeError, "kernel launch failed with status %d; device retries are disabled", status);
  return nullptr;
}

// (x, positions, inv_freq, halves, inverse, amplitude, out)
PyObject* call_rotary(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || launch_rotary == nullptr) Py_RETURN_FALSE;
  const Tensor *x = tensor_of(arguments[0]), *positions = tensor_of(arguments[1]), *inv_freq = tensor_of(arguments[2]), *out = tensor_of(arguments[6]);
  latent_rotary_call c = {};
  if (x == nullptr || positions == nullptr || inv_freq == nullptr || out == nullptr || !x->is_cuda()) Py_RETURN_FALSE;
  if (!flag_of(arguments[3], &c.layout) || !flag_of(arguments[4], &c.inverse) || !amplitude_of(arguments[5], &c.amplitude)) Py_RETURN_FALSE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  c.type = type_of(*x);
  if (c.type < 0 || (x->dim() != 2 && x->dim() != 3) || !on_device(*x, device, x->scalar_type()) || !on_device(*out, device, x->scalar_type())) Py_RETURN_FALSE;
  if (out->sizes() != x->sizes() || !rows_aligned(*x) || !rows_aligned(*out) || !entries_apart(*out)) Py_RETURN_FALSE;
  const int64_t last = x->dim() - 1;
  c.tokens = x->size(0);
  c.heads = last == 2 ? x->size(1) : 1;
  c.features = x->size(last);
  c.positions64 = positions->scalar_type() == at::kLong;
  if (inv_freq->dim() != 1) Py_RETURN_FALSE;
  c.pairs = inv_freq->size(0);
  if (!plain(*positions, device, c.positions64 ? at::kLong : at::kInt, {c.tokens}) || !plain(*inv_freq, device, at::kDouble, {c.pairs})) Py_RETURN_FALSE;
  if (c.pairs < 8 || c.pairs > LATENT_MOST_PAIRS || c.pairs % 8 != 0 || 2 * c.pairs > c.features || c.features % 8 != 0 || c.features > 65536 ||
      c.heads > 65536 || c.tokens * c.heads > kMostRows)
    Py_RETURN_FALSE;
  c.x_token = stride_of(*x, 0);
  c.out_token = stride_of(*out, 0);
  c.x_head = last == 2 ? stride_of(*x, 1) : 0;
  c.out_head = last == 2 ? stride_of(*out, 1) : 0;
  c.x = memory(*x);
  c.out = memory(*out);
  const bool in_place = c.x == c.out && c.x_token == c.out_token && c.x_head == c.out_head;
  if ((!in_place && !disjoint(*x, *out)) || !disjoint(*positions, *out) || !disjoint(*inv_freq, *out)) Py_RETURN_FALSE;
  if (x->numel() == 0) Py_RETURN_TRUE;  // (the strides of what has no entries count for nothing)
  c.positions = memory(*positions);
  c.inv_freq = memory_as<double>(*inv_freq);
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
    used_on(stream, {x, positions, inv_freq, out});
    status = launch_rotary(stream.stream(), &c);
  }
  return finished(status, {out});
  END_HANDLE_TH_ERRORS
}

// What the paged calls have in common.
struct Paged {
  int64_t batches, pages, blocks, page_rows, width;
};
bool paged(const Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, int device, at::ScalarType type, Paged* p) {
  if (cache.dim() != 4 || table.dim() != 2) return false;
  *p = {table.size(0), table.size(1), cache.size(0), cache.size(1), cache.size(3)};
  if (p->page_rows < 64 || p->page_rows % 64 != 0 || p->blocks > (INT32_MAX - 128) / p->page_rows || p->batches > INT32_MAX / 2 || p->pages > (INT32_MAX - 128) / p->page_rows) return false;
  return plain(cache, device, type, {p->blocks, p->page_rows, 1, p->width}) && rows_aligned(cache) && plain(table, device, at::kInt, {p->batches, p->pages}) &&
         plain(cu, device, at::kInt, {p->batches + 1}) && plain(lengths, device, at::kInt, {p->batches});
}

// (latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude)
PyObject* call_append(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 9 || launch_append == nullptr) Py_RETURN_FALSE;
  std::array<const Tensor*, 7> t;
  for (int i = 0; i < 7; ++i)
    if ((t[i] = tensor_of(arguments[i])) == nullptr) Py_RETURN_FALSE;
  latent_append_call c = {};
  if (!flag_of(arguments[7], &c.layout) || !amplitude_of(arguments[8], &c.amplitude) || !t[0]->is_cuda()) Py_RETURN_FALSE;
  const Tensor &latent = *t[0], &rope = *t[1], &cache = *t[2], &inv_freq = *t[6];
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = latent.scalar_type();
  c.type = type_of(latent);
  Paged p;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || latent.dim() != 2 || rope.dim() != 2 || inv_freq.dim() != 1) Py_RETURN_FALSE;
  if (!on_device(latent, device, type) || !on_device(rope, device, type) || !paged(cache, *t[3], *t[4], *t[5], device, type, &p)) Py_RETURN_FALSE;
  c.tokens = latent.size(0);
  c.pairs = inv_freq.size(0);
  if (c.pairs < 8 || c.pairs > LATENT_MOST_PAIRS || c.pairs % 8 != 0 || !plain(inv_freq, device, at::kDouble, {c.pairs})) Py_RETURN_FALSE;
  if (rope.size(0) != c.tokens || rope.size(1) != 2 * c.pairs || latent.size(1) + 2 * c.pairs != p.width || p.width % 8 != 0 || p.width > 65536 ||
      c.tokens > kMostRows || !rows_aligned(latent) || (c.tokens > 0 && rope.stride(1) != 1))
    Py_RETURN_FALSE;
  for (int i = 0; i < 7; ++i)
    if (i != 2 && !disjoint(*t[i], cache)) Py_RETURN_FALSE;
  c.latent = memory(latent);
  c.rope = memory(rope);
  c.cache = memory(cache);
  c.block_table = memory_as<int32_t>(*t[3]);
  c.cu_seqlens_q = memory_as<int32_t>(*t[4]);
  c.seqused_kv = memory_as<int32_t>(*t[5]);
  c.inv_freq = memory_as<double>(inv_freq);
  c.latent_token = latent.size(1) > 0 ? stride_of(latent, 0) : 0;
  c.rope_token = stride_of(rope, 0);
  c.batches = p.batches;
  c.pages = p.pages;
  c.blocks = p.blocks;
  c.page_rows = p.page_rows;
  c.width = p.width;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
    used_on(stream, {t[0], t[1], t[2], t[3], t[4], t[5], t[6]});
    Tensor kept;
    void* block = nullptr;
    status = int(ascendflow_host::status_block(stream, &kept, &block));
    c.status = static_cast<int32_t*>(block);
    if (status == 0) status = launch_append(stream.stream(), &c);
  }
  return finished(status, {&cache});
  END_HANDLE_TH_ERRORS
}

// (q, cache, block_table, cu_seqlens_q, seqused_kv, scale, sinks or None, out, lse or None)
PyObject* call_attention(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 9 || launch_attention == nullptr) Py_RETURN_FALSE;
  std::array<const Tensor*, 5> t;
  for (int i = 0; i < 5; ++i)
    if ((t[i] = tensor_of(arguments[i])) == nullptr) Py_RETURN_FALSE;
  const Tensor *sinks, *out = tensor_of(arguments[7]), *lse;
  latent_attention_call c = {};
  if (!number_of(arguments[5], &c.scale) || c.scale < kLeastScale || c.scale > kMostScale || out == nullptr || !optional_of(arguments[6], &sinks) || !optional_of(arguments[8], &lse) ||
      !t[0]->is_cuda())
    Py_RETURN_FALSE;
  const Tensor &q = *t[0], &cache = *t[1];
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = q.scalar_type();
  c.type = type_of(q);
  Paged p;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || q.dim() != 3 || !paged(cache, *t[2], *t[3], *t[4], device, type, &p)) Py_RETURN_FALSE;
  c.tokens = q.size(0);
  c.heads = q.size(1);
  if ((p.width != 512 && p.width != 576) || c.heads < 1 || c.tokens > kMostRows / c.heads || !plain(q, device, type, {c.tokens, c.heads, p.width}) ||
      !rows_aligned(q) || !plain(*out, device, type, {c.tokens, c.heads, LATENT_VALUES}) || !rows_aligned(*out))
    Py_RETURN_FALSE;
  if (sinks != nullptr && (!plain(*sinks, device, at::kFloat, {c.heads}) || !disjoint(*sinks, *out) || (lse != nullptr && !disjoint(*sinks, *lse)))) Py_RETURN_FALSE;
  if (lse != nullptr && (!plain(*lse, device, at::kFloat, {c.tokens, c.heads}) || !disjoint(*lse, *out))) Py_RETURN_FALSE;
  for (const Tensor* input : t)
    if (!disjoint(*input, *out) || (lse != nullptr && !disjoint(*input, *lse))) Py_RETURN_FALSE;
  c.q = memory(q);
  c.cache = memory(cache);
  c.block_table = memory_as<int32_t>(*t[2]);
  c.cu_seqlens_q = memory_as<int32_t>(*t[3]);
  c.seqused_kv = memory_as<int32_t>(*t[4]);
  c.sinks = sinks != nullptr ? memory_as<float>(*sinks) : nullptr;
  c.out = memory(*out);
  c.lse = lse != nullptr ? memory_as<float>(*lse) : nullptr;
  c.batches = p.batches;
  c.width = p.width;
  c.pages = p.pages;
  c.blocks = p.blocks;
  c.page_rows = p.page_rows;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
    used_on(stream, {t[0], t[1], t[2], t[3], t[4], sinks, out, lse});
    // Scratch of this call alone, from the allocator's pool of this stream (or of the graph that is being captured).
    uint64_t bytes = 0;
    status = workspace_size(&bytes);
    Tensor kept, scratch;
    void* block = nullptr;
    if (status == 0 && c.tokens > 0) {
      scratch = at::empty({int64_t(bytes)}, at::TensorOptions(at::kByte).device(at::kCUDA, device));
      c.workspace = scratch.mutable_data_ptr();
    }
    if (status == 0) status = int(ascendflow_host::status_block(stream, &kept, &block));
    c.status = static_cast<int32_t*>(block);
    if (status == 0) status = launch_attention(stream.stream(), &c);
  }
  return finished(status, {out, lse});
  END_HANDLE_TH_ERRORS
}

// (q, k, v, k_rope, cu_seqlens_q, cu_seqlens_k, scale, causal, out, lse or None)
PyObject* call_prefill(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 10 || launch_prefill == nullptr) Py_RETURN_FALSE;
  std::array<const Tensor*, 6> t;
  for (int i = 0; i < 6; ++i)
    if ((t[i] = tensor_of(arguments[i])) == nullptr) Py_RETURN_FALSE;
  const Tensor *out = tensor_of(arguments[8]), *lse;
  latent_prefill_call c = {};
  if (!number_of(arguments[6], &c.scale) || c.scale < kLeastScale || c.scale > kMostScale || !flag_of(arguments[7], &c.causal) || out == nullptr || !optional_of(arguments[9], &lse) ||
      !t[0]->is_cuda())
    Py_RETURN_FALSE;
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &rope = *t[3];
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = q.scalar_type();
  c.type = type_of(q);
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || q.dim() != 3 || k.dim() != 3 || t[4]->dim() != 1) Py_RETURN_FALSE;
  c.tokens = q.size(0);
  c.heads = q.size(1);
  c.keys = k.size(0);
  c.batches = t[4]->size(0) - 1;
  if (c.heads < 1 || c.heads > 65535 || c.batches < 0 || c.batches > INT32_MAX / 2 || c.tokens > kMostRows / c.heads || c.keys > kMostRows ||
      (c.tokens / 256 + c.batches) * c.heads > INT32_MAX)
    Py_RETURN_FALSE;
  if (!shaped(q, {c.tokens, c.heads, LATENT_NOPE + LATENT_ROPE}) || !shaped(k, {c.keys, c.heads, LATENT_NOPE}) || !shaped(v, {c.keys, c.heads, LATENT_NOPE}) ||
      !shaped(rope, {c.keys, LATENT_ROPE}))
    Py_RETURN_FALSE;
  for (int i = 0; i < 4; ++i)
    if (!on_device(*t[i], device, type) || !rows_aligned(*t[i]) || (t[i]->size(0) > 1 && t[i]->stride(0) == 0)) Py_RETURN_FALSE;
  if (!plain(*t[4], device, at::kInt, {c.batches + 1}) || !plain(*t[5], device, at::kInt, {c.batches + 1}) ||
      !plain(*out, device, type, {c.tokens, c.heads, LATENT_NOPE}) || !rows_aligned(*out))
    Py_RETURN_FALSE;
  if (lse != nullptr && (!plain(*lse, device, at::kFloat, {c.tokens, c.heads}) || !disjoint(*lse, *out))) Py_RETURN_FALSE;
  for (const Tensor* input : t)
    if (!disjoint(*input, *out) || (lse != nullptr && !disjoint(*input, *lse))) Py_RETURN_FALSE;
  c.q = memory(q);
  c.k = memory(k);
  c.v = memory(v);
  c.k_rope = memory(rope);
  c.cu_seqlens_q = memory_as<int32_t>(*t[4]);
  c.cu_seqlens_k = memory_as<int32_t>(*t[5]);
  c.out = memory(*out);
  c.lse = lse != nullptr ? memory_as<float>(*lse) : nullptr;
  c.q_token = stride_of(q, 0);
  c.q_head = stride_of(q, 1);
  c.k_token = stride_of(k, 0);
  c.k_head = stride_of(k, 1);
  c.v_token = stride_of(v, 0);
  c.v_head = stride_of(v, 1);
  c.rope_token = stride_of(rope, 0);
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
    used_on(stream, {t[0], t[1], t[2], t[3], t[4], t[5], out, lse});
    uint64_t bytes = 0;
    status = prefill_workspace_size(&bytes, &c);
    Tensor kept, scratch;  // (scratch: of this call alone, as above)
    void* block = nullptr;
    if (status == 0 && bytes > 0) {
      scratch = at::empty({int64_t(bytes)}, at::TensorOptions(at::kByte).device(at::kCUDA, device));
      c.workspace = scratch.mutable_data_ptr();
    }
    if (status == 0) status = int(ascendflow_host::status_block(stream, &kept, &block));
    c.status = static_cast<int32_t*>(block);
    if (status == 0) status = launch_prefill(stream.stream(), &c);
  }
  return finished(status, {out, lse});
  END_HANDLE_TH_ERRORS
}

// Addresses of the C ABI's functions, in the order in which they are declared; the class of real numbers.
PyObject* configure(PyObject*, PyObject* arguments) {
  unsigned long long rotary, append, attention, prefill, workspace, prefill_workspace;
  PyObject* real;
  if (!PyArg_ParseTuple(arguments, "KKKKKKO", &rotary, &append, &attention, &prefill, &workspace, &prefill_workspace, &real)) return nullptr;
  Py_XSETREF(real_numbers, Py_NewRef(real));
  launch_rotary = reinterpret_cast<decltype(launch_rotary)>(rotary);
  launch_append = reinterpret_cast<decltype(launch_append)>(append);
  launch_attention = reinterpret_cast<decltype(launch_attention)>(attention);
  launch_prefill = reinterpret_cast<decltype(launch_prefill)>(prefill);
  workspace_size = reinterpret_cast<decltype(workspace_size)>(workspace);
  prefill_workspace_size = reinterpret_cast<decltype(prefill_workspace_size)>(prefill_workspace);
  Py_RETURN_NONE;
}

template <PyObject* (*function)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)); }

}  // namespace

PyMethodDef ascendflow_host::latent_methods[] = {
    {"configure_latent", configure, METH_VARARGS, nullptr},
    {"rotary", fast<call_rotary>(), METH_FASTCALL, nullptr},
    {"latent_append", fast<call_append>(), METH_FASTCALL, nullptr},
    {"latent_attention", fast<call_attention>(), METH_FASTCALL, nullptr},
    {"latent_prefill", fast<call_prefill>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
