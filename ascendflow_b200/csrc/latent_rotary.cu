// Rotary positions: the queries' rope part, and a step's new rows on their way into the paged cache.
//
// y1 = a (x1 cos t - x2 sin t), y2 = a (x1 sin t + x2 cos t) with t = position * inv_freq[pair], in FP32, rounded once.
// Angles are formed as fractions of a turn in 64-bit whole numbers (`turns_of`), so far positions cost nothing
// and lose nothing; cosine and sine come from the fraction directly.
#include "latent_common.cuh"

#include <algorithm>

namespace latent {
namespace {

constexpr int kThreads = 256;

// Eight elements in 16-byte aligned memory.
template <typename T> struct Words { static constexpr int kCount = 8 * int(sizeof(T)) / 16; };
template <typename T>
__device__ __forceinline__ void load8(const T* at, uint4 (&words)[Words<T>::kCount]) {
#pragma unroll
  for (int i = 0; i < Words<T>::kCount; ++i) words[i] = reinterpret_cast<const uint4*>(at)[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* at, const uint4 (&words)[Words<T>::kCount]) {
#pragma unroll
  for (int i = 0; i < Words<T>::kCount; ++i) reinterpret_cast<uint4*>(at)[i] = words[i];
}

struct RotaryParams {
  latent_rotary_call c;
  int tokens_per_block, rotated_units, units;  // of a head: units that are turned, and besides of eight copied features
};

// A block takes a few whole tokens: their angles are worked out once for all heads. A thread turns 16 bytes of a head and, where pairs are of
// halves, the 16 bytes that go with them (or copies eight features of its part in front), of several tokens with their loads in flight
// together. Bound by memory: 8192 tokens of 64 heads and 64 features (134 MB) take 25.7 us from and to contiguous memory (5.2 TB/s), 30.7 out of
// a projection of 192 features per head into queries of 576, where every 128 bytes lie apart (no sector is read or written twice in either; cold
// launches of half as many tokens take 14.2 and 15.0). (32 bytes per thread and more blocks than run at
// once: 27.4 and 31.4.)
constexpr int kBlocks = 4;  // per SM
template <typename T, bool kHalves>
__global__ void __launch_bounds__(kThreads, kBlocks) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 turn[];  // [tokens_per_block][pairs]
  const latent_rotary_call& c = p.c;
  const int pairs = int(c.pairs);
  sm100::wait_for_predecessor();
  sm100::let_successor_start();
  const int64_t first = int64_t(blockIdx.x) * p.tokens_per_block;
  const int tokens = int(min(int64_t(p.tokens_per_block), c.tokens - first));
  for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const int64_t token = first + i / pairs;
    const int64_t position = c.positions64 ? static_cast<const int64_t*>(c.positions)[token] : static_cast<const int32_t*>(c.positions)[token];
    const uint64_t turns = turns_of(c.inv_freq[i % pairs]);
    turn[i] = turn_of(c.inverse ? -position : position, turns, float(c.amplitude));
  }
  __syncthreads();
  const int per_token = int(c.heads) * p.units, front = int(c.features) - 2 * pairs;
  const int groups = max(1, kThreads / per_token);  // tokens side by side
  const int group = groups == 1 ? 0 : int(threadIdx.x) / per_token;
  if (group >= groups) return;
  for (int i = int(threadIdx.x) - group * per_token; i < per_token; i += kThreads) {
    const int head = i / p.units, unit = i - head * p.units;
    const T* x = static_cast<const T*>(c.x) + (first + group) * c.x_token + head * c.x_head;
    T* out = static_cast<T*>(c.out) + (first + group) * c.out_token + head * c.out_head;
    const int64_t x_step = groups * c.x_token, out_step = groups * c.out_token;
    if (unit >= p.rotated_units) {
      const int at = (unit - p.rotated_units) * 8;
      for (int token = group; token < tokens; token += groups, x += x_step, out += out_step) {
#pragma unroll
        for (int k = 0; k < int(8 * sizeof(T) / 16); ++k)
          reinterpret_cast<uint4*>(out + at)[k] = reinterpret_cast<const uint4*>(x + at)[k];
      }
      continue;
    }
    const int low = front + unit * 8, high = low + pairs;
    constexpr int kInFlight = (kHalves ? 2 : 4) * 2 / int(sizeof(T));
    for (int token = group; token < tokens; token += kInFlight * groups, x += kInFlight * x_step, out += kInFlight * out_step) {
      uint4 low_words[kInFlight][Words<T>::kCount], high_words[kInFlight][Words<T>::kCount];
#pragma unroll
      for (int n = 0; n < kInFlight; ++n) {
        if (token + n * groups >= tokens) break;
        load8(x + n * x_step + low, low_words[n]);
        if constexpr (kHalves) load8(x + n * x_step + high, high_words[n]);
      }
#pragma unroll
      for (int n = 0; n < kInFlight; ++n) {
        if (token + n * groups >= tokens) break;
        const float2* angle = turn + (token + n * groups) * pairs + unit * (kHalves ? 8 : 4);
        T* a = reinterpret_cast<T*>(low_words[n]);
        T* b = reinterpret_cast<T*>(high_words[n]);
#pragma unroll
        for (int k = 0; k < (kHalves ? 8 : 4); ++k) {
          T& u = kHalves ? a[k] : a[2 * k];
          T& v = kHalves ? b[k] : a[2 * k + 1];
          const float2 t = angle[k];
          const float x1 = to_float(u), x2 = to_float(v);
          u = from_float<T>(x1 * t.x - x2 * t.y);
          v = from_float<T>(x1 * t.y + x2 * t.x);
        }
        store8(out + n * out_step + low, low_words[n]);
        if constexpr (kHalves) store8(out + n * out_step + high, high_words[n]);
      }
    }
  }
}

// One warp per new row: 8192 rows (19 MB) take 6 us with their launch, as one row does.
template <typename T, bool kHalves>
__global__ void __launch_bounds__(kThreads) append_kernel(const latent_append_call c) {
  const int lane = threadIdx.x & 31;
  sm100::wait_for_predecessor();
  sm100::let_successor_start();
  const int64_t token = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (token >= c.tokens) return;
  const int request = request_of(c.cu_seqlens_q, int(c.batches), int(token));
  if (request < 0) return;
  // (the request's tokens as the attention calls see them: offsets outside of the call's tokens are clamped)
  const int begin = bounded(c.cu_seqlens_q[request], int(c.tokens)), count = bounded(c.cu_seqlens_q[request + 1], int(c.tokens)) - begin;
  const int64_t position = int64_t(c.seqused_kv[request]) - count + (token - begin);
  const int64_t column = position / c.page_rows;
  int64_t page = -1;
  if (position >= 0 && column < c.pages) page = c.block_table[request * c.pages + column];
  if (page < 0 || page >= c.blocks) {  // nowhere to put it: reported, not written
    if (lane == 0) report(c.status, SPARSE_MLA_STATUS_BAD_PAGE, int(token), int(position));
    return;
  }
  const int pairs = int(c.pairs), front = int(c.width) - 2 * pairs;
  T* target = static_cast<T*>(c.cache) + (page * c.page_rows + position % c.page_rows) * c.width;
  const T* latent = static_cast<const T*>(c.latent) + token * c.latent_token;
  for (int at = lane * 8; at < front; at += 256) *reinterpret_cast<uint4*>(target + at) = *reinterpret_cast<const uint4*>(latent + at);
  const T* rope = static_cast<const T*>(c.rope) + token * c.rope_token;
  for (int i = lane; i < pairs; i += 32) {
    const float2 t = turn_of(position, turns_of(c.inv_freq[i]), float(c.amplitude));
    const int low = kHalves ? i : 2 * i, high = kHalves ? i + pairs : 2 * i + 1;
    const float u = to_float(rope[low]), v = to_float(rope[high]);
    target[front + low] = from_float<T>(u * t.x - v * t.y);
    target[front + high] = from_float<T>(u * t.y + v * t.x);
  }
}

template <typename T>
int launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  const int64_t blocks = (p.c.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  const size_t bytes = size_t(p.tokens_per_block) * size_t(p.c.pairs) * sizeof(float2);
  auto* kernel = p.c.layout ? rotary_kernel<T, true> : rotary_kernel<T, false>;
  return int(sm100::launch_overlapped(kernel, int(blocks), kThreads, bytes, stream, p));
}

template <typename T>
int launch_append(const latent_append_call& c, cudaStream_t stream) {
  const int64_t blocks = (c.tokens + kThreads / 32 - 1) / (kThreads / 32);
  return int(sm100::launch_overlapped(c.layout ? append_kernel<T, true> : append_kernel<T, false>, int(blocks), kThreads, 0, stream, c));
}

bool pairs_fit(int64_t pairs) { return pairs >= 8 && pairs <= LATENT_MOST_PAIRS && pairs % 8 == 0; }

}  // namespace
}  // namespace latent

extern "C" {

int launch_latent_rotary(void* stream, const latent_rotary_call* call) {
  using namespace latent;
  if (call == nullptr) return -1;
  const latent_rotary_call& c = *call;
  const int size = c.type == LATENT_F32 ? 4 : 2;
  if (c.type < LATENT_F16 || c.type > LATENT_F32 || !pairs_fit(c.pairs) || c.features < 2 * c.pairs || c.features % 8 != 0) return -1;
  if (c.tokens < 0 || c.tokens > INT32_MAX || c.heads < 0 || c.heads > 65536 || c.features > 65536) return -1;
  for (const int64_t stride : {c.x_token, c.x_head, c.out_token, c.out_head})
    if (stride * size % 16 != 0) return -1;
  if (!aligned(c.x) || !aligned(c.out) || !fits_float(c.amplitude)) return -1;
  if (c.tokens == 0 || c.heads == 0) return 0;
  RotaryParams p = {c, 1, int(c.layout ? c.pairs / 8 : c.pairs / 4), 0};
  p.units = p.rotated_units + (c.x == c.out ? 0 : int(c.features - 2 * c.pairs) / 8);
  const int64_t per_token = c.heads * p.units;  // 2^29 at most
  // All blocks run at once where there are enough tokens; tokens with few units share a block. Angles take 32 KiB at most.
  const int64_t together = kThreads / per_token, resident = int64_t(multiprocessors()) * kBlocks;
  p.tokens_per_block = int(std::min<int64_t>(std::max<int64_t>({1, together, (c.tokens + resident - 1) / resident}), 4096 / c.pairs));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.type == LATENT_F32 ? launch_rotary<float>(p, s) : c.type == LATENT_BF16 ? launch_rotary<__nv_bfloat16>(p, s) : launch_rotary<__half>(p, s);
}

int launch_latent_append(void* stream, const latent_append_call* call) {
  using namespace latent;
  if (call == nullptr) return -1;
  const latent_append_call& c = *call;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || !pairs_fit(c.pairs) || c.width < 2 * c.pairs || c.width % 8 != 0 || c.width > 65536) return -1;
  if (c.batches < 0 || c.batches >= INT32_MAX || c.tokens < 0 || c.tokens > INT32_MAX || c.pages < 0 || c.blocks < 0 || c.page_rows < 1) return -1;
  if (!aligned(c.latent) || c.latent_token % 8 != 0 || !aligned(c.cache) || !fits_float(c.amplitude) || c.status == nullptr) return -1;
  if (c.tokens == 0 || c.batches == 0) return 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.type == LATENT_BF16 ? launch_append<__nv_bfloat16>(c, s) : launch_append<__half>(c, s);
}

}  // extern "C"
