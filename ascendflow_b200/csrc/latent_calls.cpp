// The host side of the operators around dense latent attention: checks and launches, as host_calls.cpp does them for
// the sparse operator. A call that passes is launched through the C ABI and the function returns True; for one that does
// not it returns False without having enqueued anything, and `latent.py` finds the violated rule and words the error.

#include "call_checks.h"

#include <ATen/ops/empty.h>

#include <cmath>
#include <limits>

namespace {

using namespace ascendflow_host;

decltype(&launch_latent_rotary) launch_rotary = nullptr;
decltype(&launch_latent_append) launch_append = nullptr;
decltype(&launch_latent_attention) launch_attention = nullptr;
decltype(&launch_latent_prefill) launch_prefill = nullptr;
decltype(&launch_latent_append8) launch_append8 = nullptr;
decltype(&launch_latent_attention8) launch_attention8 = nullptr;
decltype(&workspace_size_latent_attention) workspace_size = nullptr;
decltype(&workspace_size_latent_prefill) prefill_workspace_size = nullptr;

// What FP32 holds; for scales with room to spare. (No NaN.)
bool amplitude_fits(double value) { return std::abs(value) <= std::numeric_limits<float>::max(); }
bool scale_fits(double value) { return value >= 1e-30 && value <= 1e30; }
constexpr int64_t kMostRows = int64_t(1) << 30;  // tokens x heads

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

// Scales of a cache held in 8 bits, [blocks, page_rows / rows that share one].
bool scaled(const Tensor& scales, const Paged& p, int device, int64_t* block_rows) {
  if (!scales.defined() || scales.dim() != 2 || scales.size(1) < 1 || p.page_rows % scales.size(1) != 0) return false;
  *block_rows = p.page_rows / scales.size(1);
  return *block_rows <= 64 && (*block_rows & (*block_rows - 1)) == 0 && plain(scales, device, at::kFloat8_e8m0fnu, {p.blocks, scales.size(1)});
}

// `scales`: those of a cache held in 8 bits.
int append(const Tensor& latent, const Tensor& rope, const Tensor& cache, const Tensor* scales, const Tensor& table, const Tensor& cu, const Tensor& lengths, const Tensor& inv_freq,
           bool halves, double amplitude) {
  if (launch_append == nullptr || !latent.defined() || !latent.is_cuda() || !rope.defined() || !inv_freq.defined() || !amplitude_fits(amplitude)) return kRefused;
  latent_append_call c = {};
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = latent.scalar_type();
  c.layout = halves;
  c.amplitude = amplitude;
  c.type = type_of(latent);
  Paged p;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || latent.dim() != 2 || rope.dim() != 2 || inv_freq.dim() != 1) return kRefused;
  if (!on_device(latent, device, type) || !on_device(rope, device, type) || !paged(cache, table, cu, lengths, device, scales != nullptr ? at::kFloat8_e4m3fn : type, &p))
    return kRefused;
  int64_t block_rows = 0;
  if (scales != nullptr && (!scaled(*scales, p, device, &block_rows) || p.width % 16 != 0 || p.batches > (1 << 26))) return kRefused;
  c.tokens = latent.size(0);
  c.pairs = inv_freq.size(0);
  if (c.pairs < 8 || c.pairs > LATENT_MOST_PAIRS || c.pairs % 8 != 0 || !plain(inv_freq, device, at::kDouble, {c.pairs})) return kRefused;
  if (rope.size(0) != c.tokens || rope.size(1) != 2 * c.pairs || latent.size(1) + 2 * c.pairs != p.width || p.width % 8 != 0 || p.width > 65536 ||
      c.tokens > kMostRows || !rows_aligned(latent) || (c.tokens > 0 && rope.stride(1) != 1))
    return kRefused;
  for (const Tensor* t : {&latent, &rope, &table, &cu, &lengths, &inv_freq})
    if (!disjoint(*t, cache) || (scales != nullptr && !disjoint(*t, *scales))) return kRefused;
  if (scales != nullptr && !disjoint(cache, *scales)) return kRefused;
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
  used_on(stream, {&latent, &rope, &cache, scales, &table, &cu, &lengths, &inv_freq});
  Tensor kept;
  void* block = nullptr;
  if (const cudaError_t error = ascendflow_host::status_block(stream, &kept, &block)) return int(error);
  c.status = static_cast<int32_t*>(block);
  if (scales != nullptr) {
    const latent_append8_call call = {c, memory_as<uint8_t>(*scales), block_rows};
    return launch_append8(stream.stream(), &call);
  }
  return launch_append(stream.stream(), &c);
}

int attention(const Tensor& q, const Tensor& cache, const Tensor* scales, const Tensor& table, const Tensor& cu, const Tensor& lengths, double scale, const Tensor* sinks,
              const Tensor& out, const Tensor* lse) {
  if (launch_attention == nullptr || !q.defined() || !q.is_cuda() || !scale_fits(scale)) return kRefused;
  latent_attention_call c = {};
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::ScalarType type = q.scalar_type();
  c.scale = scale;
  c.type = type_of(q);
  Paged p;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || q.dim() != 3 || !paged(cache, table, cu, lengths, device, scales != nullptr ? at::kFloat8_e4m3fn : type, &p))
    return kRefused;
  int64_t block_rows = 0;
  if (scales != nullptr && (!scaled(*scales, p, device, &block_rows) || !disjoint(*scales, out) || (lse != nullptr && !disjoint(*scales, *lse)))) return kRefused;
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
  used_on(stream, {&q, &cache, scales, &table, &cu, &lengths, sinks, &out, lse});
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
  if (scales != nullptr) {
    const latent_attention8_call call = {c, memory_as<const uint8_t>(*scales), block_rows};
    return launch_attention8(stream.stream(), &call);
  }
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

// (latent, rope, cache, [scales,] block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude)
template <bool kHeld8>
PyObject* call_append(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  constexpr int more = kHeld8;
  std::array<const Tensor*, 7 + more> t;
  bool halves;
  double amplitude;
  if (count != 9 + more || !tensors_of(arguments, &t) || !flag_of(arguments[7 + more], &halves) || !number_of(arguments[8 + more], &amplitude)) Py_RETURN_FALSE;
  const Tensor* scales = kHeld8 ? t[3] : nullptr;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = append(*t[0], *t[1], *t[2], scales, *t[3 + more], *t[4 + more], *t[5 + more], *t[6 + more], halves, amplitude);
  }
  return finished(status, {t[2], scales});
  END_HANDLE_TH_ERRORS
}

// (q, cache, [scales,] block_table, cu_seqlens_q, seqused_kv, scale, sinks or None, out, lse or None)
template <bool kHeld8>
PyObject* call_attention(PyObject*, PyObject* const* arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  constexpr int more = kHeld8;
  std::array<const Tensor*, 5 + more> t;
  const Tensor *sinks, *lse;
  double scale;
  if (count != 9 + more || !tensors_of(arguments, &t) || !number_of(arguments[5 + more], &scale) || !optional_of(arguments[6 + more], &sinks) ||
      !optional_of(arguments[8 + more], &lse))
    Py_RETURN_FALSE;
  const Tensor* out = tensor_of(arguments[7 + more]);
  if (out == nullptr) Py_RETURN_FALSE;
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = attention(*t[0], *t[1], kHeld8 ? t[2] : nullptr, *t[2 + more], *t[3 + more], *t[4 + more], scale, sinks, *out, lse);
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

const Tensor* given(const std::optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

void rotary_op(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, bool halves, bool inverse, double amplitude, Tensor& out) {
  settle(rotary(x, positions, inv_freq, halves, inverse, amplitude, out), "rotary",
         {boxed(x), boxed(positions), boxed(inv_freq), boxed(halves), boxed(inverse), boxed(amplitude), boxed(out)});
}
void append_op(const Tensor& latent, const Tensor& rope, Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, const Tensor& inv_freq, bool halves,
               double amplitude) {
  settle(append(latent, rope, cache, nullptr, table, cu, lengths, inv_freq, halves, amplitude), "latent_append",
         {boxed(latent), boxed(rope), boxed(cache), boxed(table), boxed(cu), boxed(lengths), boxed(inv_freq), boxed(halves), boxed(amplitude)});
}
void attention_op(const Tensor& q, const Tensor& cache, const Tensor& table, const Tensor& cu, const Tensor& lengths, double scale, const std::optional<Tensor>& sinks, Tensor& out,
                  const std::optional<Tensor>& lse) {
  settle(attention(q, cache, nullptr, table, cu, lengths, scale, given(sinks), out, given(lse)), "latent_attention",
         {boxed(q), boxed(cache), boxed(table), boxed(cu), boxed(lengths), boxed(scale), boxed(sinks), boxed(out), boxed(lse)});
}
void append8_op(const Tensor& latent, const Tensor& rope, Tensor& cache, Tensor& scales, const Tensor& table, const Tensor& cu, const Tensor& lengths, const Tensor& inv_freq, bool halves,
                double amplitude) {
  settle(append(latent, rope, cache, &scales, table, cu, lengths, inv_freq, halves, amplitude), "latent_append8",
         {boxed(latent), boxed(rope), boxed(cache), boxed(scales), boxed(table), boxed(cu), boxed(lengths), boxed(inv_freq), boxed(halves), boxed(amplitude)});
}
void attention8_op(const Tensor& q, const Tensor& cache, const Tensor& scales, const Tensor& table, const Tensor& cu, const Tensor& lengths, double scale,
                   const std::optional<Tensor>& sinks, Tensor& out, const std::optional<Tensor>& lse) {
  settle(attention(q, cache, &scales, table, cu, lengths, scale, given(sinks), out, given(lse)), "latent_attention8",
         {boxed(q), boxed(cache), boxed(scales), boxed(table), boxed(cu), boxed(lengths), boxed(scale), boxed(sinks), boxed(out), boxed(lse)});
}
void prefill_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& rope, const Tensor& cu_q, const Tensor& cu_k, double scale, bool causal, Tensor& out,
                const std::optional<Tensor>& lse) {
  settle(prefill(q, k, v, rope, cu_q, cu_k, scale, causal, out, given(lse)), "latent_prefill",
         {boxed(q), boxed(k), boxed(v), boxed(rope), boxed(cu_q), boxed(cu_k), boxed(scale), boxed(causal), boxed(out), boxed(lse)});
}

TORCH_LIBRARY_FRAGMENT(ascendflow_b200, m) {
  const std::vector<at::Tag> tags = {at::Tag::pt2_compliant_tag};
  m.def("rotary(Tensor x, Tensor positions, Tensor inv_freq, bool halves, bool inverse, float amplitude, Tensor(a!) out) -> ()", tags);
  m.def("latent_append(Tensor latent, Tensor rope, Tensor(a!) cache, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, Tensor inv_freq, bool halves, "
        "float amplitude) -> ()", tags);
  m.def("latent_attention(Tensor q, Tensor cache, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, float scale, Tensor? sinks, Tensor(a!) out, "
        "Tensor(b!)? lse) -> ()", tags);
  m.def("latent_append8(Tensor latent, Tensor rope, Tensor(a!) cache, Tensor(b!) scales, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, Tensor inv_freq, "
        "bool halves, float amplitude) -> ()", tags);
  m.def("latent_attention8(Tensor q, Tensor cache, Tensor scales, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, float scale, Tensor? sinks, Tensor(a!) out, "
        "Tensor(b!)? lse) -> ()", tags);
  m.def("latent_prefill(Tensor q, Tensor k, Tensor v, Tensor k_rope, Tensor cu_seqlens_q, Tensor cu_seqlens_k, float scale, bool causal, Tensor(a!) out, "
        "Tensor(b!)? lse) -> ()", tags);
}
TORCH_LIBRARY_IMPL(ascendflow_b200, CUDA, m) {
  m.impl("rotary", rotary_op);
  m.impl("latent_append", append_op);
  m.impl("latent_attention", attention_op);
  m.impl("latent_prefill", prefill_op);
  m.impl("latent_append8", append8_op);
  m.impl("latent_attention8", attention8_op);
}
constexpr const char* kNames[] = {"rotary", "latent_append", "latent_attention", "latent_prefill", "latent_append8", "latent_attention8"};
TORCH_LIBRARY_IMPL(ascendflow_b200, ADInplaceOrView, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&mutates>());
}
TORCH_LIBRARY_IMPL(ascendflow_b200, Autograd, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&without_gradient>());
}

// Addresses of the C ABI's functions, in the order in which they are declared; the class of real numbers.
PyObject* configure(PyObject*, PyObject* arguments) {
  unsigned long long rotary, append, attention, prefill, workspace, prefill_workspace, append8, attention8;
  PyObject* real;
  if (!PyArg_ParseTuple(arguments, "KKKKKKKKO", &rotary, &append, &attention, &prefill, &workspace, &prefill_workspace, &append8, &attention8, &real)) return nullptr;
  Py_XSETREF(real_numbers, Py_NewRef(real));
  launch_rotary = reinterpret_cast<decltype(launch_rotary)>(rotary);
  launch_append = reinterpret_cast<decltype(launch_append)>(append);
  launch_attention = reinterpret_cast<decltype(launch_attention)>(attention);
  launch_prefill = reinterpret_cast<decltype(launch_prefill)>(prefill);
  launch_append8 = reinterpret_cast<decltype(launch_append8)>(append8);
  launch_attention8 = reinterpret_cast<decltype(launch_attention8)>(attention8);
  workspace_size = reinterpret_cast<decltype(workspace_size)>(workspace);
  prefill_workspace_size = reinterpret_cast<decltype(prefill_workspace_size)>(prefill_workspace);
  Py_RETURN_NONE;
}

// The front end's call for what the registered ops refuse.
PyObject* set_fallback(PyObject*, PyObject* function) {
  Py_XSETREF(checked_call, Py_NewRef(function));
  Py_RETURN_NONE;
}

}  // namespace

PyMethodDef ascendflow_host::latent_methods[] = {
    {"configure_latent", configure, METH_VARARGS, nullptr},
    {"set_latent_fallback", set_fallback, METH_O, nullptr},
    {"rotary", fast<call_rotary>(), METH_FASTCALL, nullptr},
    {"latent_append", fast<call_append<false>>(), METH_FASTCALL, nullptr},
    {"latent_attention", fast<call_attention<false>>(), METH_FASTCALL, nullptr},
    {"latent_prefill", fast<call_prefill>(), METH_FASTCALL, nullptr},
    {"latent_append8", fast<call_append<true>>(), METH_FASTCALL, nullptr},
    {"latent_attention8", fast<call_attention<true>>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
