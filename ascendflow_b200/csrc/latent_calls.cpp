// The host side of the operators around dense latent attention: checks and launches, as host_calls.cpp does them for
// the sparse operator. A call that passes is launched through the C ABI and the function returns True; for one that does
// not it returns False without having enqueued anything, and `latent.py` finds the violated rule and words the error.

#include "host_calls.h"

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <functional>
#include <limits>
#include <optional>
#include <vector>

#include "../../include/latent.h"

namespace {

using Tensor = at::Tensor;

decltype(&launch_latent_rotary) launch_rotary = nullptr;
decltype(&launch_latent_append) launch_append = nullptr;
decltype(&launch_latent_attention) launch_attention = nullptr;
decltype(&launch_latent_prefill) launch_prefill = nullptr;
decltype(&workspace_size_latent_attention) workspace_size = nullptr;
decltype(&workspace_size_latent_prefill) prefill_workspace_size = nullptr;

// What FP32 holds; for scales with room to spare. (No NaN.)
bool amplitude_fits(double value) { return std::abs(value) <= std::numeric_limits<float>::max(); }
bool scale_fits(double value) { return value >= 1e-30 && value <= 1e30; }
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
  return true;
}
bool flag_of(PyObject* object, bool* value) {
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

PyObject* raise_launch_status(int status) {
  PyErr_Format(PyExc_RuntimeError, "kernel launch failed with status %d; device retries are disabled", status);
  return nullptr;
}
// What was written in place counts its version up, as for any in-place operation (a tensor made in inference mode has none).
void count_up(const Tensor* t) {
  if (t != nullptr && t->defined() && !t->is_inference()) torch::autograd::increment_version(*t);
}

// Each call: checks and launch. kRefused: not accepted, nothing enqueued; otherwise the launch's status.
constexpr int kRefused = -1000;

int rotary(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, bool halves, bool inverse, double amplitude, const Tensor& out) {
  if (launch_rotary == nullptr || !x.defined() || !x.is_cuda() || !out.defined() || !positions.defined() || !amplitude_fits(amplitude)) return kRefused;
  latent_rotary_call c = {};
  const c10::DeviceIndex device = c10::cuda::current_device();
  c.layout = halves;
  c.inverse = inverse;
  c.amplitude = amplitude;
  c.type = type_of(x);
  if (c.type < 0 || (x.dim() != 2 && x.dim() != 3) || !on_device(x, device, x.scalar_type()) || !on_device(out, device, x.scalar_type())) return kRefused;
  if (out.sizes() != x.sizes() || !rows_aligned(x) || !rows_aligned(out) || !entries_apart(out)) return kRefused;
  const int64_t last = x.dim() - 1;
  c.tokens = x.size(0);
  c.heads = last == 2 ? x.size(1) : 1;
  c.features = x.size(last);
  c.positions64 = positions.scalar_type() == at::kLong;
  if (!inv_freq.defined() || inv_freq.dim() != 1) return kRefused;
  c.pairs = inv_freq.size(0);
  if (!plain(positions, device, c.positions64 ? at::kLong : at::kInt, {c.tokens}) || !plain(inv_freq, device, at::kDouble, {c.pairs})) return kRefused;
  if (c.pairs < 8 || c.pairs > LATENT_MOST_PAIRS || c.pairs % 8 != 0 || 2 * c.pairs > c.features || c.features % 8 != 0 || c.features > 65536 ||
      c.heads > 65536 || c.tokens * c.heads > kMostRows)
    return kRefused;
  c.x_token = stride_of(x, 0);
  c.out_token = stride_of(out, 0);
  c.x_head = last == 2 ? stride_of(x, 1) : 0;
  c.out_head = last == 2 ? stride_of(out, 1) : 0;
  c.x = memory(x);
  c.out = memory(out);
  const bool in_place = c.x == c.out && c.x_token == c.out_token && c.x_head == c.out_head;
  if ((!in_place && !disjoint(x, out)) || !disjoint(positions, out) || !disjoint(inv_freq, out)) return kRefused;
  if (x.numel() == 0) return 0;  // (the strides of what has no entries count for nothing)
  c.positions = memory(positions);
  c.inv_freq = memory_as<double>(inv_freq);
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&x, &positions, &inv_freq, &out});
  return launch_rotary(stream.stream(), &c);
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

int append(const Tensor& latent, const Tensor& rope, const Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, const Tensor& inv_freq, bool halves,
           double amplitude) {
  if (launch_append == nullptr || !latent.defined() || !latent.is_cuda() || !rope.defined() || !inv_freq.defined() || !amplitude_fits(amplitude)) return kRefused;
  latent_append_call c = {};
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = latent.scalar_type();
  c.layout = halves;
  c.amplitude = amplitude;
  c.type = type_of(latent);
  Paged p;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || latent.dim() != 2 || rope.dim() != 2 || inv_freq.dim() != 1) return kRefused;
  if (!on_device(latent, device, type) || !on_device(rope, device, type) || !paged(cache, table, cu, lengths, device, type, &p)) return kRefused;
  c.tokens = latent.size(0);
  c.pairs = inv_freq.size(0);
  if (c.pairs < 8 || c.pairs > LATENT_MOST_PAIRS || c.pairs % 8 != 0 || !plain(inv_freq, device, at::kDouble, {c.pairs})) return kRefused;
  if (rope.size(0) != c.tokens || rope.size(1) != 2 * c.pairs || latent.size(1) + 2 * c.pairs != p.width || p.width % 8 != 0 || p.width > 65536 ||
      c.tokens > kMostRows || !rows_aligned(latent) || (c.tokens > 0 && rope.stride(1) != 1))
    return kRefused;
  for (const Tensor* t : {&latent, &rope, &table, &cu, &lengths, &inv_freq})
    if (!disjoint(*t, cache)) return kRefused;
  c.latent = memory(latent);
  c.rope = memory(rope);
  c.cache = memory(cache);
  c.block_table = memory_as<int32_t>(table);
  c.cu_seqlens_q = memory_as<int32_t>(cu);
  c.seqused_kv = memory_as<int32_t>(lengths);
  c.inv_freq = memory_as<double>(inv_freq);
  c.latent_token = latent.size(1) > 0 ? stride_of(latent, 0) : 0;
  c.rope_token = stride_of(rope, 0);
  c.batches = p.batches;
  c.pages = p.pages;
  c.blocks = p.blocks;
  c.page_rows = p.page_rows;
  c.width = p.width;
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&latent, &rope, &cache, &table, &cu, &lengths, &inv_freq});
  Tensor kept;
  void* block = nullptr;
  if (const cudaError_t error = ascendflow_host::status_block(stream, &kept, &block)) return int(error);
  c.status = static_cast<int32_t*>(block);
  return launch_append(stream.stream(), &c);
}

int attention(const Tensor& q, const Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, double scale, const Tensor* sinks, const Tensor& out,
              const Tensor* lse) {
  if (launch_attention == nullptr || !q.defined() || !q.is_cuda() || !scale_fits(scale)) return kRefused;
  latent_attention_call c = {};
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = q.scalar_type();
  c.scale = scale;
  c.type = type_of(q);
  Paged p;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || q.dim() != 3 || !paged(cache, table, cu, lengths, device, type, &p)) return kRefused;
  c.tokens = q.size(0);
  c.heads = q.size(1);
  if ((p.width != 512 && p.width != 576) || c.heads < 1 || c.tokens > kMostRows / c.heads || !plain(q, device, type, {c.tokens, c.heads, p.width}) ||
      !rows_aligned(q) || !plain(out, device, type, {c.tokens, c.heads, LATENT_VALUES}) || !rows_aligned(out))
    return kRefused;
  if (sinks != nullptr && (!plain(*sinks, device, at::kFloat, {c.heads}) || !disjoint(*sinks, out) || (lse != nullptr && !disjoint(*sinks, *lse)))) return kRefused;
  if (lse != nullptr && (!plain(*lse, device, at::kFloat, {c.tokens, c.heads}) || !disjoint(*lse, out))) return kRefused;
  for (const Tensor* input : {&q, &cache, &table, &cu, &lengths})
    if (!disjoint(*input, out) || (lse != nullptr && !disjoint(*input, *lse))) return kRefused;
  c.q = memory(q);
  c.cache = memory(cache);
  c.block_table = memory_as<int32_t>(table);
  c.cu_seqlens_q = memory_as<int32_t>(cu);
  c.seqused_kv = memory_as<int32_t>(lengths);
  c.sinks = sinks != nullptr ? memory_as<float>(*sinks) : nullptr;
  c.out = memory(out);
  c.lse = lse != nullptr ? memory_as<float>(*lse) : nullptr;
  c.batches = p.batches;
  c.width = p.width;
  c.pages = p.pages;
  c.blocks = p.blocks;
  c.page_rows = p.page_rows;
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&q, &cache, &table, &cu, &lengths, sinks, &out, lse});
  // Scratch of this call alone, from the allocator's pool of this stream (or of the graph that is being captured).
  uint64_t bytes = 0;
  if (const int status = workspace_size(&bytes)) return status;
  Tensor kept, scratch;
  void* block = nullptr;
  if (c.tokens > 0) {
    scratch = at::empty({int64_t(bytes)}, at::TensorOptions(at::kByte).device(at::kCUDA, device));
    c.workspace = scratch.mutable_data_ptr();
  }
  if (const cudaError_t error = ascendflow_host::status_block(stream, &kept, &block)) return int(error);
  c.status = static_cast<int32_t*>(block);
  return launch_attention(stream.stream(), &c);
}

int prefill(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& rope, const Tensor& cu_q, const Tensor& cu_k, double scale, bool causal, const Tensor& out,
            const Tensor* lse) {
  if (launch_prefill == nullptr || !q.defined() || !q.is_cuda() || !k.defined() || !v.defined() || !rope.defined() || !cu_q.defined() || !scale_fits(scale)) return kRefused;
  latent_prefill_call c = {};
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = q.scalar_type();
  c.scale = scale;
  c.causal = causal;
  c.type = type_of(q);
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || q.dim() != 3 || k.dim() != 3 || cu_q.dim() != 1) return kRefused;
  c.tokens = q.size(0);
  c.heads = q.size(1);
  c.keys = k.size(0);
  c.batches = cu_q.size(0) - 1;
  if (c.heads < 1 || c.heads > 65535 || c.batches < 0 || c.batches > INT32_MAX / 2 || c.tokens > kMostRows / c.heads || c.keys > kMostRows ||
      (c.tokens / 256 + c.batches) * c.heads > INT32_MAX)
    return kRefused;
  if (!shaped(q, {c.tokens, c.heads, LATENT_NOPE + LATENT_ROPE}) || !shaped(k, {c.keys, c.heads, LATENT_NOPE}) || !shaped(v, {c.keys, c.heads, LATENT_NOPE}) ||
      !shaped(rope, {c.keys, LATENT_ROPE}))
    return kRefused;
  for (const Tensor* t : {&q, &k, &v, &rope})
    if (!on_device(*t, device, type) || !rows_aligned(*t) || (t->size(0) > 1 && t->stride(0) == 0)) return kRefused;
  if (!plain(cu_q, device, at::kInt, {c.batches + 1}) || !plain(cu_k, device, at::kInt, {c.batches + 1}) ||
      !plain(out, device, type, {c.tokens, c.heads, LATENT_NOPE}) || !rows_aligned(out))
    return kRefused;
  if (lse != nullptr && (!plain(*lse, device, at::kFloat, {c.tokens, c.heads}) || !disjoint(*lse, out))) return kRefused;
  for (const Tensor* input : {&q, &k, &v, &rope, &cu_q, &cu_k})
    if (!disjoint(*input, out) || (lse != nullptr && !disjoint(*input, *lse))) return kRefused;
  c.q = memory(q);
  c.k = memory(k);
  c.v = memory(v);
  c.k_rope = memory(rope);
  c.cu_seqlens_q = memory_as<int32_t>(cu_q);
  c.cu_seqlens_k = memory_as<int32_t>(cu_k);
  c.out = memory(out);
  c.lse = lse != nullptr ? memory_as<float>(*lse) : nullptr;
  c.q_token = stride_of(q, 0);
  c.q_head = stride_of(q, 1);
  c.k_token = stride_of(k, 0);
  c.k_head = stride_of(k, 1);
  c.v_token = stride_of(v, 0);
  c.v_head = stride_of(v, 1);
  c.rope_token = stride_of(rope, 0);
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&q, &k, &v, &rope, &cu_q, &cu_k, &out, lse});
  uint64_t bytes = 0;
  if (const int status = prefill_workspace_size(&bytes, &c)) return status;
  Tensor kept, scratch;  // (scratch: of this call alone, as above)
  void* block = nullptr;
  if (bytes > 0) {
    scratch = at::empty({int64_t(bytes)}, at::TensorOptions(at::kByte).device(at::kCUDA, device));
    c.workspace = scratch.mutable_data_ptr();
  }
  if (const cudaError_t error = ascendflow_host::status_block(stream, &kept, &block)) return int(error);
  c.status = static_cast<int32_t*>(block);
  return launch_prefill(stream.stream(), &c);
}

// ---- Python functions --------------------------------------------------------------------------------

// True, False for a refused call, or an error.
PyObject* finished(int status, std::initializer_list<const Tensor*> written) {
  if (status == kRefused) Py_RETURN_FALSE;
  if (status != 0) return raise_launch_status(status);
  for (const Tensor* t : written) count_up(t);
  Py_RETURN_TRUE;
}

// Plain tensors in the first arguments, and nobody who wants to see what is called (a dispatch mode, as in tracing; the front end then calls the registered op).
template <size_t N>
bool tensors_of(PyObject* const* arguments, std::array<const Tensor*, N>* tensors) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
  for (size_t i = 0; i < N; ++i)
    if (((*tensors)[i] = tensor_of(arguments[i])) == nullptr) return false;
  return true;
}

// (x, positions, inv_freq, halves, inverse, amplitude, out)
PyObject* call_rotary(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::array<const Tensor*, 3> t;
  bool halves, inverse;
  double amplitude;
  if (count != 7 || !tensors_of(arguments, &t) || !flag_of(arguments[3], &halves) || !flag_of(arguments[4], &inverse) || !number_of(arguments[5], &amplitude)) Py_RETURN_FALSE;
  const Tensor* out = tensor_of(arguments[6]);
  if (out == nullptr) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;  // the caller holds references to all of them
    status = rotary(*t[0], *t[1], *t[2], halves, inverse, amplitude, *out);
  }
  return finished(status, {out});
  END_HANDLE_TH_ERRORS
}

// (latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude)
PyObject* call_append(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::array<const Tensor*, 7> t;
  bool halves;
  double amplitude;
  if (count != 9 || !tensors_of(arguments, &t) || !flag_of(arguments[7], &halves) || !number_of(arguments[8], &amplitude)) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = append(*t[0], *t[1], *t[2], *t[3], *t[4], *t[5], *t[6], halves, amplitude);
  }
  return finished(status, {t[2]});
  END_HANDLE_TH_ERRORS
}

// (q, cache, block_table, cu_seqlens_q, seqused_kv, scale, sinks or None, out, lse or None)
PyObject* call_attention(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::array<const Tensor*, 5> t;
  const Tensor *sinks, *lse;
  double scale;
  if (count != 9 || !tensors_of(arguments, &t) || !number_of(arguments[5], &scale) || !optional_of(arguments[6], &sinks) || !optional_of(arguments[8], &lse)) Py_RETURN_FALSE;
  const Tensor* out = tensor_of(arguments[7]);
  if (out == nullptr) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = attention(*t[0], *t[1], *t[2], *t[3], *t[4], scale, sinks, *out, lse);
  }
  return finished(status, {out, lse});
  END_HANDLE_TH_ERRORS
}

// (q, k, v, k_rope, cu_seqlens_q, cu_seqlens_k, scale, causal, out, lse or None)
PyObject* call_prefill(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::array<const Tensor*, 6> t;
  const Tensor* lse;
  bool causal;
  double scale;
  if (count != 10 || !tensors_of(arguments, &t) || !number_of(arguments[6], &scale) || !flag_of(arguments[7], &causal) || !optional_of(arguments[9], &lse)) Py_RETURN_FALSE;
  const Tensor* out = tensor_of(arguments[8]);
  if (out == nullptr) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = prefill(*t[0], *t[1], *t[2], *t[3], *t[4], *t[5], scale, causal, *out, lse);
  }
  return finished(status, {out, lse});
  END_HANDLE_TH_ERRORS
}

// ---- the registered ops ------------------------------------------------------------------------------

PyObject* checked_call = nullptr;  // the front end's call, for arguments refused here

// What the launch said; a refused call goes through the front end, (name, arguments ...), which words the error.
void settle(int status, const char* name, std::initializer_list<std::function<PyObject*()>> arguments) {
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
auto boxed(const Tensor& t) {
  return [&t] { return THPVariable_Wrap(t); };
}
auto boxed(const std::optional<Tensor>& t) {
  return [&t] { return t.has_value() ? THPVariable_Wrap(*t) : Py_NewRef(Py_None); };
}
auto boxed(double value) {
  return [value] { return PyFloat_FromDouble(value); };
}
auto boxed(bool value) {
  return [value] { return PyBool_FromLong(value); };
}
const Tensor* given(const std::optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

void rotary_op(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, bool halves, bool inverse, double amplitude, Tensor& out) {
  settle(rotary(x, positions, inv_freq, halves, inverse, amplitude, out), "rotary",
         {boxed(x), boxed(positions), boxed(inv_freq), boxed(halves), boxed(inverse), boxed(amplitude), boxed(out)});
}
void append_op(const Tensor& latent, const Tensor& rope, Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, const Tensor& inv_freq, bool halves,
               double amplitude) {
  settle(append(latent, rope, cache, table, cu, lengths, inv_freq, halves, amplitude), "latent_append",
         {boxed(latent), boxed(rope), boxed(cache), boxed(table), boxed(cu), boxed(lengths), boxed(inv_freq), boxed(halves), boxed(amplitude)});
}
void attention_op(const Tensor& q, const Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, double scale, const std::optional<Tensor>& sinks, Tensor& out,
                  const std::optional<Tensor>& lse) {
  settle(attention(q, cache, table, cu, lengths, scale, given(sinks), out, given(lse)), "latent_attention",
         {boxed(q), boxed(cache), boxed(table), boxed(cu), boxed(lengths), boxed(scale), boxed(sinks), boxed(out), boxed(lse)});
}
void prefill_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& rope, const Tensor& cu_q, const Tensor& cu_k, double scale, bool causal, Tensor& out,
                const std::optional<Tensor>& lse) {
  settle(prefill(q, k, v, rope, cu_q, cu_k, scale, causal, out, given(lse)), "latent_prefill",
         {boxed(q), boxed(k), boxed(v), boxed(rope), boxed(cu_q), boxed(cu_k), boxed(scale), boxed(causal), boxed(out), boxed(lse)});
}

// No gradient: tensors that want one are refused, also while a graph is traced.
void without_gradient(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  if (at::GradMode::is_enabled())
    for (const c10::IValue& argument : torch::jit::last(*stack, op.schema().arguments().size()))
      TORCH_CHECK(!argument.isTensor() || !argument.toTensor().defined() || !argument.toTensor().requires_grad(), op.schema().name(), ": the operator has no gradient");
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

// What is written in place counts its version up.
void mutates(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const auto& parameters = op.schema().arguments();
  const auto arguments = torch::jit::last(*stack, parameters.size());
  std::vector<Tensor> written;
  for (size_t i = 0; i < parameters.size(); ++i)
    if (parameters[i].alias_info() != nullptr && parameters[i].alias_info()->isWrite() && arguments[i].isTensor()) written.push_back(arguments[i].toTensor());
  {
    at::AutoDispatchBelowADInplaceOrView below;
    op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
  }
  for (const Tensor& t : written) count_up(&t);
}

TORCH_LIBRARY_FRAGMENT(ascendflow_b200, m) {
  const std::vector<at::Tag> tags = {at::Tag::pt2_compliant_tag};
  m.def("rotary(Tensor x, Tensor positions, Tensor inv_freq, bool halves, bool inverse, float amplitude, Tensor(a!) out) -> ()", tags);
  m.def("latent_append(Tensor latent, Tensor rope, Tensor(a!) cache, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, Tensor inv_freq, bool halves, "
        "float amplitude) -> ()", tags);
  m.def("latent_attention(Tensor q, Tensor cache, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, float scale, Tensor? sinks, Tensor(a!) out, "
        "Tensor(b!)? lse) -> ()", tags);
  m.def("latent_prefill(Tensor q, Tensor k, Tensor v, Tensor k_rope, Tensor cu_seqlens_q, Tensor cu_seqlens_k, float scale, bool causal, Tensor(a!) out, "
        "Tensor(b!)? lse) -> ()", tags);
}
TORCH_LIBRARY_IMPL(ascendflow_b200, CUDA, m) {
  m.impl("rotary", rotary_op);
  m.impl("latent_append", append_op);
  m.impl("latent_attention", attention_op);
  m.impl("latent_prefill", prefill_op);
}
constexpr const char* kNames[] = {"rotary", "latent_append", "latent_attention", "latent_prefill"};
TORCH_LIBRARY_IMPL(ascendflow_b200, ADInplaceOrView, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&mutates>());
}
TORCH_LIBRARY_IMPL(ascendflow_b200, Autograd, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&without_gradient>());
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

// The front end's call for what the registered ops refuse.
PyObject* set_fallback(PyObject*, PyObject* function) {
  Py_XSETREF(checked_call, Py_NewRef(function));
  Py_RETURN_NONE;
}

template <PyObject* (*function)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)); }

}  // namespace

PyMethodDef ascendflow_host::latent_methods[] = {
    {"configure_latent", configure, METH_VARARGS, nullptr},
    {"set_latent_fallback", set_fallback, METH_O, nullptr},
    {"rotary", fast<call_rotary>(), METH_FASTCALL, nullptr},
    {"latent_append", fast<call_append>(), METH_FASTCALL, nullptr},
    {"latent_attention", fast<call_attention>(), METH_FASTCALL, nullptr},
    {"latent_prefill", fast<call_prefill>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
