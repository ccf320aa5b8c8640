// Attention over the paged latent cache in absorbed form: one row per token is key and value of all heads.
#include "latent_common.cuh"

namespace latent {
namespace {

// One warp per token and head: running maximum and sum, a key at a time.
template <typename T, int kWidth>
__global__ void __launch_bounds__(256) attention_kernel(const latent_attention_call c) {
  constexpr int kOwn = kWidth / 32, kOwnValues = LATENT_VALUES / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= c.tokens * c.heads) return;
  const int token = int(row / c.heads), head = int(row % c.heads);
  const int request = request_of(c.cu_seqlens_q, int(c.batches), token);
  if (request < 0) return;
  const int begin = c.cu_seqlens_q[request], count = c.cu_seqlens_q[request + 1] - begin;
  const int keys = c.seqused_kv[request] - count + (token - begin) + 1;
  const float scale = float(c.scale) * 1.4426950408889634f;
  float q[kOwn], o[kOwnValues] = {};
#pragma unroll
  for (int i = 0; i < kOwn; ++i) q[i] = to_float(static_cast<const T*>(c.q)[row * kWidth + i * 32 + lane]) * scale;
  float most = -INFINITY, sum = 0.f;
  for (int key = 0; key < keys; ++key) {
    const int64_t column = key / c.page_rows;
    const int64_t page = column < c.pages ? c.block_table[request * c.pages + column] : -1;
    if (page < 0 || page >= c.blocks) {
      if (lane == 0) report(c.status, SPARSE_MLA_STATUS_BAD_PAGE, token, key);
      continue;
    }
    const T* k = static_cast<const T*>(c.cache) + (page * c.page_rows + key % c.page_rows) * kWidth + lane;
    float values[kOwn], score = 0.f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) score += q[i] * (values[i] = to_float(k[i * 32]));
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) score += __shfl_xor_sync(0xffffffffu, score, i);
    const float next = fmaxf(most, score), alpha = exp2f(most - next), weight = exp2f(score - next);
    most = next;
    sum = sum * alpha + weight;
#pragma unroll
    for (int i = 0; i < kOwnValues; ++i) o[i] = o[i] * alpha + weight * values[i];
  }
  float inverse = sum > 0.f ? 1.f / sum : 0.f, log_sum = sum > 0.f ? most + log2f(sum) : -INFINITY;
  const float sink = c.sinks != nullptr ? c.sinks[head] * 1.4426950408889634f : -INFINITY, top = fmaxf(log_sum, sink);
  if (sink > -INFINITY) {
    const float total = exp2f(log_sum - top) + exp2f(sink - top);
    inverse = sum > 0.f ? inverse * exp2f(log_sum - top) / total : 0.f;
    log_sum = top + log2f(total);
  }
  T* out = static_cast<T*>(c.out) + row * LATENT_VALUES + lane;
#pragma unroll
  for (int i = 0; i < kOwnValues; ++i) out[i * 32] = from_float<T>(o[i] * inverse);
  if (c.lse != nullptr && lane == 0) c.lse[row] = log_sum * 0.6931471805599453f;
}

}  // namespace
}  // namespace latent

extern "C" {

int workspace_size_latent_attention(uint64_t* bytes) {
  if (bytes == nullptr) return -1;
  *bytes = 512;
  return 0;
}

int launch_latent_attention(void* stream, const latent_attention_call* call) {
  using namespace latent;
  const latent_attention_call& c = *call;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || (c.width != 512 && c.width != 576)) return -1;
  if (c.batches < 0 || c.tokens < 0 || c.heads < 1 || c.pages < 0 || c.blocks < 0 || c.page_rows < 64 || c.page_rows % 64 != 0) return -1;
  if (c.tokens == 0 || c.batches == 0) return 0;
  auto* kernel = c.type == LATENT_BF16 ? (c.width == 576 ? attention_kernel<__nv_bfloat16, 576> : attention_kernel<__nv_bfloat16, 512>)
                                       : (c.width == 576 ? attention_kernel<__half, 576> : attention_kernel<__half, 512>);
  kernel<<<unsigned((c.tokens * c.heads + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(c);
  return int(cudaGetLastError());
}

}  // extern "C"
