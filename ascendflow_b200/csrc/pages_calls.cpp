// The host side of the operators on the pages of a cache: checks and launches, as latent_calls.cpp does them (a refused call returns False, and
// `pages.py` words the error).

#include "call_checks.h"

#include <ATen/ops/empty.h>

#include "../../include/pages.h"

namespace {

using namespace ascendflow_host;

decltype(&launch_pages_resize) launch_resize = nullptr;
decltype(&launch_pages_fork) launch_fork = nullptr;
decltype(&launch_pages_compact) launch_compact = nullptr;
decltype(&workspace_size_pages_resize) resize_workspace = nullptr;
decltype(&workspace_size_pages_fork) fork_workspace = nullptr;
decltype(&workspace_size_pages_compact) compact_workspace = nullptr;

// The same tensor's memory, or none of it.
bool same_or_disjoint(const Tensor& a, const Tensor& b) { return (a.const_data_ptr() == b.const_data_ptr() && a.sizes() == b.sizes()) || disjoint(a, b); }

// What the calls have in common.
bool described(pages_call* c, const Tensor& table, const Tensor& counts, const Tensor* lengths, int64_t page_rows, const Tensor& counts_out, int device) {
  if (!table.defined() || !counts.defined() || !counts_out.defined() || table.dim() != 2 || counts.dim() != 1 || page_rows < 1 || page_rows > INT32_MAX) return false;
  c->requests = table.size(0);
  c->entries = table.size(1);
  c->blocks = counts.size(0);
  c->page_rows = page_rows;
  if (c->blocks > PAGES_MOST_BLOCKS || c->requests >= INT32_MAX || c->entries >= INT32_MAX || table.numel() > INT32_MAX) return false;
  if (!plain(table, device, at::kInt, {c->requests, c->entries}) || !plain(counts, device, at::kInt, {c->blocks}) || !plain(counts_out, device, at::kInt, {c->blocks}) ||
      !same_or_disjoint(counts, counts_out) || !disjoint(table, counts) || !disjoint(table, counts_out))
    return false;
  c->table_in = memory_as<int32_t>(table);
  c->counts_in = memory_as<int32_t>(counts);
  c->counts_out = memory_as<int32_t>(counts_out);
  if (lengths == nullptr) return true;
  c->lengths = memory_as<int32_t>(*lengths);
  return plain(*lengths, device, at::kInt, {c->requests}) && disjoint(*lengths, counts_out);
}

// Caches of `blocks` pages, of `page_rows` cached rows or a divisor of them each (compact: of anything), none overlapping with another nor with `others`.
bool described(std::vector<pages_tensor>* found, at::TensorList caches, int64_t blocks, int64_t page_rows, int device, std::initializer_list<const Tensor*> others) {
  if (caches.size() > PAGES_MOST_TENSORS) return false;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  for (const Tensor& cache : caches) {
    if (!cache.defined() || cache.dim() < (page_rows > 0 ? 2 : 1) || !on_device(cache, device, cache.scalar_type()) || !cache.is_contiguous() || cache.size(0) != blocks) return false;
    const int64_t rows = page_rows > 0 ? cache.size(1) : 1;
    if (rows < 1 || (page_rows > 0 && page_rows % rows != 0)) return false;
    found->push_back({memory(cache), blocks > 0 ? int64_t(cache.nbytes()) / blocks : 0, rows});
    for (const Tensor* other : others)
      if (!disjoint(cache, *other)) return false;
    if (cache.numel() > 0) spans.push_back(span(cache));
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return false;
  return true;
}

// Scratch of this call alone, from the allocator's pool of this stream (or of the graph that is being captured), and the block that reports go to.
struct Kept {
  Tensor scratch, status;
};
int prepare(pages_call* c, uint64_t bytes, const c10::cuda::CUDAStream& stream, Kept* kept) {
  kept->scratch = at::empty({int64_t(bytes)}, at::TensorOptions(at::kByte).device(at::kCUDA, stream.device_index()));
  c->workspace = kept->scratch.mutable_data_ptr();
  void* block = nullptr;
  if (const cudaError_t error = status_block(stream, &kept->status, &block)) return int(error);
  c->status = static_cast<int32_t*>(block);
  return 0;
}

int resize(const Tensor& table, const Tensor& counts, const Tensor& lengths, int64_t page_rows, const Tensor& table_out, const Tensor& counts_out) {
  if (launch_resize == nullptr || !table.defined() || !table.is_cuda() || !lengths.defined() || !table_out.defined()) return kRefused;
  const c10::DeviceIndex device = c10::cuda::current_device();
  pages_call c = {};
  if (!described(&c, table, counts, &lengths, page_rows, counts_out, device) || !plain(table_out, device, at::kInt, {c.requests, c.entries})) return kRefused;
  if (!same_or_disjoint(table, table_out) || !disjoint(lengths, table_out) || !disjoint(counts, table_out) || !disjoint(counts_out, table_out)) return kRefused;
  c.table_out = memory_as<int32_t>(table_out);
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&table, &counts, &lengths, &table_out, &counts_out});
  uint64_t bytes = 0;
  Kept kept;
  if (const int status = resize_workspace(&bytes, &c)) return status;
  if (const int status = prepare(&c, bytes, stream, &kept)) return status;
  return launch_resize(stream.stream(), &c);
}

int fork(at::TensorList caches, const Tensor& table, const Tensor& counts, const Tensor& parents, const Tensor& lengths, int64_t page_rows, const Tensor& table_out,
         const Tensor& counts_out) {
  if (launch_fork == nullptr || !table.defined() || !table.is_cuda() || !lengths.defined() || !parents.defined() || !table_out.defined() || parents.dim() != 1) return kRefused;
  const c10::DeviceIndex device = c10::cuda::current_device();
  pages_fork_call c = {};
  c.children = parents.size(0);
  if (!described(&c.pages, table, counts, &lengths, page_rows, counts_out, device) || !plain(parents, device, at::kInt, {c.children}) || c.children >= INT32_MAX ||
      !plain(table_out, device, at::kInt, {c.children, c.pages.entries}) || table_out.numel() > INT32_MAX)
    return kRefused;
  for (const Tensor* t : {&table, &counts, &lengths, &parents, &counts_out})
    if (!disjoint(*t, table_out)) return kRefused;
  if (!disjoint(parents, counts_out)) return kRefused;
  std::vector<pages_tensor> tensors;
  if (!described(&tensors, caches, c.pages.blocks, page_rows, device, {&table, &counts, &lengths, &parents, &table_out, &counts_out})) return kRefused;
  c.pages.table_out = memory_as<int32_t>(table_out);
  c.parents = memory_as<int32_t>(parents);
  c.tensors = tensors.data();
  c.tensor_count = int64_t(tensors.size());
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&table, &counts, &lengths, &parents, &table_out, &counts_out});
  for (const Tensor& cache : caches) used_on(stream, {&cache});
  uint64_t bytes = 0;
  Kept kept;
  if (const int status = fork_workspace(&bytes, &c)) return status;
  if (const int status = prepare(&c.pages, bytes, stream, &kept)) return status;
  return launch_fork(stream.stream(), &c);
}

int compact(at::TensorList caches, const Tensor& table, const Tensor& counts, const Tensor& table_out, const Tensor& counts_out, const Tensor& places) {
  if (launch_compact == nullptr || !table.defined() || !table.is_cuda() || !table_out.defined() || !places.defined()) return kRefused;
  const c10::DeviceIndex device = c10::cuda::current_device();
  pages_compact_call c = {};
  if (!described(&c.pages, table, counts, nullptr, 1, counts_out, device) || !plain(table_out, device, at::kInt, {c.pages.requests, c.pages.entries}) ||
      !plain(places, device, at::kInt, {c.pages.blocks}) || !same_or_disjoint(table, table_out) || !disjoint(counts, table_out) || !disjoint(counts_out, table_out))
    return kRefused;
  for (const Tensor* t : {&table, &counts, &table_out, &counts_out})
    if (!disjoint(*t, places)) return kRefused;
  std::vector<pages_tensor> tensors;
  if (!described(&tensors, caches, c.pages.blocks, 0, device, {&table, &counts, &table_out, &counts_out, &places})) return kRefused;
  c.pages.table_out = memory_as<int32_t>(table_out);
  c.places = memory_as<int32_t>(places);
  c.tensors = tensors.data();
  c.tensor_count = int64_t(tensors.size());
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  used_on(stream, {&table, &counts, &table_out, &counts_out, &places});
  for (const Tensor& cache : caches) used_on(stream, {&cache});
  uint64_t bytes = 0;
  Kept kept;
  if (const int status = compact_workspace(&bytes, &c)) return status;
  if (const int status = prepare(&c.pages, bytes, stream, &kept)) return status;
  return launch_compact(stream.stream(), &c);
}

// ---- Python functions --------------------------------------------------------------------------------

bool whole_of(PyObject* object, int64_t* value) {
  if (!PyLong_Check(object) || PyBool_Check(object)) return false;
  int overflow = 0;
  *value = PyLong_AsLongLongAndOverflow(object, &overflow);
  return overflow == 0;
}
// A list or tuple of plain tensors.
bool list_of(PyObject* object, std::vector<Tensor>* tensors) {
  if (!PyList_Check(object) && !PyTuple_Check(object)) return false;
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(object);
  tensors->reserve(size_t(count));
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor* t = tensor_of(PySequence_Fast_GET_ITEM(object, i));
    if (t == nullptr) return false;
    tensors->push_back(*t);
  }
  return true;
}

// Outputs that are given, or new ones (an int32 tensor of `sizes` on the device of `like`) where None is.
struct Output {
  const Tensor* given = nullptr;
  Tensor made;
  bool from(PyObject* object) { return optional_of(object, &given); }
  const Tensor& tensor(const Tensor& like, at::IntArrayRef sizes) {
    if (given != nullptr) return *given;
    made = at::empty(sizes, at::TensorOptions(at::kInt).device(like.device()));
    return made;
  }
  const Tensor* written() const { return given != nullptr ? given : &made; }
};
// A tuple of the outputs, False for a refused call, or an error.
template <size_t N>
PyObject* results(int status, const std::array<Output*, N>& outs) {
  if (status == kRefused) Py_RETURN_FALSE;
  if (status != 0) return raise_launch_status(status);
  PyObject* tuple = PyTuple_New(Py_ssize_t(N));
  for (size_t i = 0; i < N; ++i) {
    count_up(outs[i]->given);
    PyTuple_SET_ITEM(tuple, Py_ssize_t(i), THPVariable_Wrap(*outs[i]->written()));
  }
  return tuple;
}
bool plain_cuda(const Tensor& t, int64_t dims) { return t.defined() && t.is_cuda() && t.dim() == dims; }

// (block_table, counts, lengths, page_rows, table_out or None, counts_out or None): (table, counts)
PyObject* call_resize(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::array<const Tensor*, 3> t;
  Output table, counts;
  int64_t page_rows;
  if (count != 6 || !tensors_of(arguments, &t) || !whole_of(arguments[3], &page_rows) || !table.from(arguments[4]) || !counts.from(arguments[5])) Py_RETURN_FALSE;
  if (!plain_cuda(*t[0], 2) || !plain_cuda(*t[1], 1)) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;  // the caller holds references to all of them
    status = resize(*t[0], *t[1], *t[2], page_rows, table.tensor(*t[0], t[0]->sizes()), counts.tensor(*t[1], t[1]->sizes()));
  }
  return results<2>(status, {&table, &counts});
  END_HANDLE_TH_ERRORS
}

// (caches, block_table, counts, parents, lengths, page_rows, table_out or None, counts_out or None): (table, counts)
PyObject* call_fork(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::vector<Tensor> caches;
  std::array<const Tensor*, 4> t;
  Output table, counts;
  int64_t page_rows;
  if (count != 8 || !list_of(arguments[0], &caches) || !tensors_of(arguments + 1, &t) || !whole_of(arguments[5], &page_rows) || !table.from(arguments[6]) || !counts.from(arguments[7]))
    Py_RETURN_FALSE;
  if (!plain_cuda(*t[0], 2) || !plain_cuda(*t[1], 1) || !plain_cuda(*t[2], 1)) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = fork(caches, *t[0], *t[1], *t[2], *t[3], page_rows, table.tensor(*t[0], {t[2]->size(0), t[0]->size(1)}), counts.tensor(*t[1], t[1]->sizes()));
  }
  if (status == 0)
    for (const Tensor& cache : caches) count_up(&cache);
  return results<2>(status, {&table, &counts});
  END_HANDLE_TH_ERRORS
}

// (caches, block_table, counts, table_out or None, counts_out or None, places or None): (table, counts, places)
PyObject* call_compact(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  std::vector<Tensor> caches;
  std::array<const Tensor*, 2> t;
  Output table, counts, places;
  if (count != 6 || !list_of(arguments[0], &caches) || !tensors_of(arguments + 1, &t) || !table.from(arguments[3]) || !counts.from(arguments[4]) || !places.from(arguments[5]))
    Py_RETURN_FALSE;
  if (!plain_cuda(*t[0], 2) || !plain_cuda(*t[1], 1)) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = compact(caches, *t[0], *t[1], table.tensor(*t[0], t[0]->sizes()), counts.tensor(*t[1], t[1]->sizes()), places.tensor(*t[1], t[1]->sizes()));
  }
  if (status == 0)
    for (const Tensor& cache : caches) count_up(&cache);
  return results<3>(status, {&table, &counts, &places});
  END_HANDLE_TH_ERRORS
}

// ---- the registered ops ------------------------------------------------------------------------------

void resize_op(const Tensor& table, const Tensor& counts, const Tensor& lengths, int64_t page_rows, Tensor& table_out, Tensor& counts_out) {
  settle(resize(table, counts, lengths, page_rows, table_out, counts_out), "pages_resize",
         {boxed(table), boxed(counts), boxed(lengths), boxed(page_rows), boxed(table_out), boxed(counts_out)});
}
void fork_op(at::TensorList caches, const Tensor& table, const Tensor& counts, const Tensor& parents, const Tensor& lengths, int64_t page_rows, Tensor& table_out, Tensor& counts_out) {
  settle(fork(caches, table, counts, parents, lengths, page_rows, table_out, counts_out), "pages_fork",
         {boxed(caches), boxed(table), boxed(counts), boxed(parents), boxed(lengths), boxed(page_rows), boxed(table_out), boxed(counts_out)});
}
void compact_op(at::TensorList caches, const Tensor& table, const Tensor& counts, Tensor& table_out, Tensor& counts_out, Tensor& places) {
  settle(compact(caches, table, counts, table_out, counts_out, places), "pages_compact",
         {boxed(caches), boxed(table), boxed(counts), boxed(table_out), boxed(counts_out), boxed(places)});
}

TORCH_LIBRARY_FRAGMENT(ascendflow_b200, m) {
  const std::vector<at::Tag> tags = {at::Tag::pt2_compliant_tag};
  m.def("pages_resize(Tensor block_table, Tensor counts, Tensor lengths, int page_rows, Tensor(a!) table_out, Tensor(b!) counts_out) -> ()", tags);
  m.def("pages_fork(Tensor(a!)[] caches, Tensor block_table, Tensor counts, Tensor parents, Tensor lengths, int page_rows, Tensor(b!) table_out, Tensor(c!) counts_out) -> ()", tags);
  m.def("pages_compact(Tensor(a!)[] caches, Tensor block_table, Tensor counts, Tensor(b!) table_out, Tensor(c!) counts_out, Tensor(d!) places) -> ()", tags);
}
TORCH_LIBRARY_IMPL(ascendflow_b200, CUDA, m) {
  m.impl("pages_resize", resize_op);
  m.impl("pages_fork", fork_op);
  m.impl("pages_compact", compact_op);
}
constexpr const char* kNames[] = {"pages_resize", "pages_fork", "pages_compact"};
TORCH_LIBRARY_IMPL(ascendflow_b200, ADInplaceOrView, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&mutates>());
}
TORCH_LIBRARY_IMPL(ascendflow_b200, Autograd, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&without_gradient>());
}

// Addresses of the C ABI's functions: the launches, then the workspace sizes.
PyObject* configure(PyObject*, PyObject* arguments) {
  unsigned long long address[6];
  if (!PyArg_ParseTuple(arguments, "KKKKKK", address, address + 1, address + 2, address + 3, address + 4, address + 5)) return nullptr;
  launch_resize = reinterpret_cast<decltype(launch_resize)>(address[0]);
  launch_fork = reinterpret_cast<decltype(launch_fork)>(address[1]);
  launch_compact = reinterpret_cast<decltype(launch_compact)>(address[2]);
  resize_workspace = reinterpret_cast<decltype(resize_workspace)>(address[3]);
  fork_workspace = reinterpret_cast<decltype(fork_workspace)>(address[4]);
  compact_workspace = reinterpret_cast<decltype(compact_workspace)>(address[5]);
  Py_RETURN_NONE;
}

}  // namespace

PyMethodDef ascendflow_host::pages_methods[] = {
    {"configure_pages", configure, METH_VARARGS, nullptr},
    {"pages_resize", fast<call_resize>(), METH_FASTCALL, nullptr},
    {"pages_fork", fast<call_fork>(), METH_FASTCALL, nullptr},
    {"pages_compact", fast<call_compact>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
