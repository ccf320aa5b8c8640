// Attention of prompts in expanded form: keys and values per head, and one rope key per token for all heads.
#include "latent_common.cuh"

namespace latent {
namespace {

// One warp per token and head: running maximum and sum, a key at a time.
template <typename T>
__global__ void __launch_bounds__(256) prefill_kernel(const latent_prefill_call c) {
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= c.tokens * c.heads) return;
  const int token = int(row % c.tokens), head = int(row / c.tokens);
  const int request = request_of(c.cu_seqlens_q, int(c.batches), token);
  if (request < 0) return;
  const int begin = c.cu_seqlens_q[request], count = c.cu_seqlens_q[request + 1] - begin;
  const int first = c.cu_seqlens_k[request], length = c.cu_seqlens_k[request + 1] - first;
  const int keys = c.causal ? length - count + (token - begin) + 1 : length;
  const float scale = float(c.scale) * 1.4426950408889634f;
  float q[6], o[4] = {};
#pragma unroll
  for (int i = 0; i < 6; ++i) q[i] = to_float(static_cast<const T*>(c.q)[token * c.q_token + head * c.q_head + i * 32 + lane]) * scale;
  float most = -INFINITY, sum = 0.f;
  for (int64_t key = first; key < first + keys; ++key) {
    const T* k = static_cast<const T*>(c.k) + key * c.k_token + head * c.k_head + lane;
    const T* v = static_cast<const T*>(c.v) + key * c.v_token + head * c.v_head + lane;
    const T* rope = static_cast<const T*>(c.k_rope) + key * c.rope_token + lane;
    float score = q[4] * to_float(rope[0]) + q[5] * to_float(rope[32]);
#pragma unroll
    for (int i = 0; i < 4; ++i) score += q[i] * to_float(k[i * 32]);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) score += __shfl_xor_sync(0xffffffffu, score, i);
    const float next = fmaxf(most, score), alpha = exp2f(most - next), weight = exp2f(score - next);
    most = next;
    sum = sum * alpha + weight;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * alpha + weight * to_float(v[i * 32]);
  }
  const float inverse = sum > 0.f ? 1.f / sum : 0.f;
  T* out = static_cast<T*>(c.out) + (int64_t(token) * c.heads + head) * LATENT_NOPE + lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i * 32] = from_float<T>(o[i] * inverse);
  if (c.lse != nullptr && lane == 0) c.lse[int64_t(token) * c.heads + head] = sum > 0.f ? (most + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace
}  // namespace latent

extern "C" int launch_latent_prefill(void* stream, const latent_prefill_call* call) {
  using namespace latent;
  const latent_prefill_call& c = *call;
  if (c.type != LATENT_F16 && c.type != LATENT_BF16) return -1;
  if (c.batches < 0 || c.tokens < 0 || c.keys < 0 || c.heads < 1) return -1;
  if (c.tokens == 0 || c.batches == 0) return 0;
  const unsigned blocks = unsigned((c.tokens * c.heads + 7) / 8);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c.type == LATENT_BF16) prefill_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(c);
  else prefill_kernel<__half><<<blocks, 256, 0, s>>>(c);
  return int(cudaGetLastError());
}
