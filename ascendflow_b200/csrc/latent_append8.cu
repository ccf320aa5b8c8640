// A step's new rows into a cache held in 8 bits: rope part turned, e4m3 numbers with a power-of-two scale for every block of rows.
//
// k = least whole number with max|v| <= 448 2^k over the block's new rows, and not below the block's own where older rows precede them; c = v 2^-k rounded
// to e4m3. As scales are powers of two, a division by one is exact: a number is rounded once (and once more where its block's scale grows and it becomes a
// subnormal one). Bound by latency: four rows to a warp, all of whose loads are on their way together, and which stay in registers between the maximum and the
// numbers (rows of more than 512 features in front or 32 pairs are read twice). A block's warps meet once. 8192 rows in blocks of 64 (14 MB) 7.1 us, 14.6
// with eight rows to a warp that were read twice.
#include "latent_common.cuh"

#include <algorithm>
#include <type_traits>

namespace latent {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kRowsPerWarp = 4;
constexpr int kMostFront = 512, kMostPairs = 32;  // of rows that registers hold
constexpr uint32_t kInfinity = 0x7f800000u, kMostHalf = 0x47700000u;  // bits of FP32 numbers: infinity, 61440

struct Append8Params {
  latent_append_call c;
  uint8_t* scales;
  int shift;  // 2^this rows share a scale
};

// Blocks of requests in front of `b` are dealt items below this: a request of n tokens touches n / G + 2 blocks of G rows at most.
__device__ __forceinline__ int64_t items_before(const Append8Params& p, int b) { return (bounded(p.c.cu_seqlens_q[b], int(p.c.tokens)) >> p.shift) + 2 * int64_t(b); }

// The scale's byte that |v| needs, from its bits: 2^(byte - 127) >= |v| / 448.
__device__ __forceinline__ int scale_for(uint32_t most) {
  if (most >= kInfinity) return 255;
  return max(int(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u), 0);
}
// Two numbers of e4m3, rounded to nearest.
__device__ __forceinline__ uint32_t numbers_of(float low, float high) {
  uint16_t pair;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(pair) : "f"(high), "f"(low));
  return pair;
}
// Two numbers of e4m3 times a power of two that is at most 1 (exact until the last rounding: half holds four bits down to 2^-21).
__device__ __forceinline__ uint32_t numbers_times(uint32_t pair, __half2 factor) {
  uint32_t wide;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(wide) : "h"(uint16_t(pair)));
  const __half2 scaled = __hmul2(reinterpret_cast<const __half2&>(wide), factor);
  uint16_t narrow;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(narrow) : "r"(reinterpret_cast<const uint32_t&>(scaled)));
  return narrow;
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude(float v) {
  const uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
  return std::is_same<T, __half>::value && bits < kInfinity ? min(bits, kMostHalf) : bits;
}
template <typename T>
__device__ __forceinline__ float cut(float v) {
  return std::is_same<T, __half>::value ? fminf(fmaxf(v, -61440.f), 61440.f) : v;
}

// A block of rows by `together` neighbouring warps of a block of threads, every together-th row by one of them.
template <typename T, bool kHalves, bool kKept>
__global__ void __launch_bounds__(kThreads) append8_kernel(const Append8Params p) {
  __shared__ uint32_t maxima[kWarps];
  const latent_append_call& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block = 1 << p.shift, together = max(block / kRowsPerWarp, 1), member = warp & (together - 1);
  sm100::wait_for_predecessor();
  sm100::let_successor_start();
  const int64_t item = (int64_t(blockIdx.x) * kWarps + warp) / together;
  const int batches = int(c.batches), pairs = int(c.pairs), front = int(c.width) - 2 * pairs;
  // Rows `older` .. rows - 1 of a block are the call's; its first row lies at `row0` of the cache and has position `base`. None: older = rows.
  int older = 0, rows = 0, begin = 0;
  int64_t base = 0, row0 = 0, start = 0;
  if (item < items_before(p, batches)) {
    int request = 0;
    for (int high = batches; high - request > 1;) {
      const int middle = (request + high) >> 1;
      if (items_before(p, middle) <= item) request = middle; else high = middle;
    }
    const int64_t which = item - items_before(p, request);
    // (the request's tokens as the attention calls see them: offsets outside of the call's tokens are clamped)
    begin = bounded(c.cu_seqlens_q[request], int(c.tokens));
    const int count = bounded(c.cu_seqlens_q[request + 1], int(c.tokens)) - begin;
    const int64_t end = c.seqused_kv[request];
    start = end - count;  // position of the request's first new row
    if (which >= 0 && count > 0) {
      if (which == 0 && start < 0 && member == 0 && lane == 0) report(c.status, SPARSE_MLA_STATUS_BAD_PAGE, begin, int(start));
      base = ((max(start, int64_t(0)) >> p.shift) + which) << p.shift;
      const int64_t first = max(max(start, int64_t(0)), base), last = min(end, base + block);
      if (first < last) {
        const int64_t column = base / c.page_rows;
        int64_t page = -1;
        if (column < c.pages) page = c.block_table[request * c.pages + column];
        if (page >= 0 && page < c.blocks) {
          row0 = page * c.page_rows + (base - column * c.page_rows);
          older = int(first - base);
          rows = int(last - base);
        } else if (member == 0 && lane == 0) {  // nowhere to put them: reported, not written
          report(c.status, SPARSE_MLA_STATUS_BAD_PAGE, int(begin + (first - start)), int(first));
        }
      }
    }
  }
  const T* latent = static_cast<const T*>(c.latent) + (begin + (base - start)) * c.latent_token;  // of the block's row 0, which may be none of the call's
  const T* rope = static_cast<const T*>(c.rope) + (begin + (base - start)) * c.rope_token;
  uint8_t* held = static_cast<uint8_t*>(c.cache) + row0 * c.width;
  auto mine = [&](int n) { return member + n * together; };
  auto is_new = [&](int n) { return mine(n) >= older && mine(n) < rows; };
  auto turned = [&](int row, int i, float u, float v) {
    const float2 t = turn_of(base + row, turns_of(c.inv_freq[i]), float(c.amplitude));
    return make_float2(u * t.x - v * t.y, u * t.y + v * t.x);
  };
  auto rope_of = [&](int row, int i) {
    const T* own = rope + row * c.rope_token;
    return make_float2(to_float(own[kHalves ? i : 2 * i]), to_float(own[kHalves ? i + pairs : 2 * i + 1]));
  };

  uint4 kept[kRowsPerWarp][2];
  float2 kept_pair[kRowsPerWarp];
  uint32_t most = 0;
  auto see = [&](const uint4& words) {
    const T* v = reinterpret_cast<const T*>(&words);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, magnitude<T>(to_float(v[e])));
  };
  if constexpr (kKept) {
#pragma unroll
    for (int n = 0; n < kRowsPerWarp; ++n) {
      kept[n][0] = kept[n][1] = make_uint4(0, 0, 0, 0);
      kept_pair[n] = make_float2(0.f, 0.f);
      if (!is_new(n)) continue;
      const T* row = latent + mine(n) * c.latent_token;
      if (lane * 8 < front) kept[n][0] = *reinterpret_cast<const uint4*>(row + lane * 8);
      if (lane * 8 + 256 < front) kept[n][1] = *reinterpret_cast<const uint4*>(row + lane * 8 + 256);
      if (lane < pairs) kept_pair[n] = rope_of(mine(n), lane);
    }
#pragma unroll
    for (int n = 0; n < kRowsPerWarp; ++n) {
      if (!is_new(n)) continue;
      see(kept[n][0]);
      see(kept[n][1]);
      if (lane < pairs) kept_pair[n] = turned(mine(n), lane, kept_pair[n].x, kept_pair[n].y);
      most = max(most, max(magnitude<T>(kept_pair[n].x), magnitude<T>(kept_pair[n].y)));
    }
  } else {
    for (int n = 0; n < kRowsPerWarp; ++n) {
      if (!is_new(n)) continue;
      for (int at = lane * 8; at < front; at += 256) see(*reinterpret_cast<const uint4*>(latent + mine(n) * c.latent_token + at));
      for (int i = lane; i < pairs; i += 32) {
        const float2 v = rope_of(mine(n), i), w = turned(mine(n), i, v.x, v.y);
        most = max(most, max(magnitude<T>(w.x), magnitude<T>(w.y)));
      }
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  uint8_t* own_scale = p.scales + (row0 >> p.shift);
  const int had = older > 0 ? *own_scale : 0;
  if (lane == 0) maxima[warp] = most;
  __syncthreads();  // (everybody has read the scale, too)
  for (int w = warp - member; w < warp - member + together; ++w) most = max(most, maxima[w]);
  if (older >= rows) return;
  const int scale = max(scale_for(most), had);
  if (member == 0 && lane == 0) *own_scale = uint8_t(scale);

  if (scale > had && scale != 255) {  // the rows in front, in terms of the new scale
    const __half2 factor = __float2half2_rn(had - scale < -24 ? 0.f : __uint_as_float(uint32_t(127 + had - scale) << 23));
    for (int row = member; row < older; row += together) {
      for (int at = lane * 8; at < int(c.width); at += 256) {
        uint2* place = reinterpret_cast<uint2*>(held + row * c.width + at);
        uint2 v = *place;
        v.x = numbers_times(v.x & 0xffffu, factor) | numbers_times(v.x >> 16, factor) << 16;
        v.y = numbers_times(v.y & 0xffffu, factor) | numbers_times(v.y >> 16, factor) << 16;
        *place = v;
      }
    }
  }
  // 1 / scale in two factors: either is a normal number
  const int half = (127 - scale) / 2, rest = 127 - scale - half;
  const float by = scale == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(uint32_t(127 + half) << 23), and_by = __uint_as_float(uint32_t(127 + rest) << 23);
  auto number = [&](float low, float high) { return numbers_of(cut<T>(low) * by * and_by, cut<T>(high) * by * and_by); };
  auto store_latent = [&](uint8_t* target, const uint4& words) {
    const T* v = reinterpret_cast<const T*>(&words);
    uint32_t pair[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) pair[e] = number(to_float(v[2 * e]), to_float(v[2 * e + 1]));
    *reinterpret_cast<uint2*>(target) = make_uint2(pair[0] | pair[1] << 16, pair[2] | pair[3] << 16);
  };
  auto store_pair = [&](uint8_t* target, int i, float2 v) {
    const uint32_t pair = number(v.x, v.y);
    if constexpr (kHalves) {
      target[front + i] = uint8_t(pair);
      target[front + i + pairs] = uint8_t(pair >> 8);
    } else {
      *reinterpret_cast<uint16_t*>(target + front + 2 * i) = uint16_t(pair);
    }
  };
#pragma unroll
  for (int n = 0; n < kRowsPerWarp; ++n) {
    if (!is_new(n)) continue;
    uint8_t* target = held + mine(n) * c.width;
    if constexpr (kKept) {
      if (lane * 8 < front) store_latent(target + lane * 8, kept[n][0]);
      if (lane * 8 + 256 < front) store_latent(target + lane * 8 + 256, kept[n][1]);
      if (lane < pairs) store_pair(target, lane, kept_pair[n]);
    } else {
      for (int at = lane * 8; at < front; at += 256) store_latent(target + at, *reinterpret_cast<const uint4*>(latent + mine(n) * c.latent_token + at));
      for (int i = lane; i < pairs; i += 32) {
        const float2 v = rope_of(mine(n), i);
        store_pair(target, i, turned(mine(n), i, v.x, v.y));
      }
    }
  }
}

template <typename T, bool kHalves>
int launch_append8(const Append8Params& p, cudaStream_t stream) {
  const int64_t items = (p.c.tokens >> p.shift) + 2 * p.c.batches, together = std::max((1 << p.shift) / kRowsPerWarp, 1);
  const bool kept = p.c.pairs <= kMostPairs && p.c.width - 2 * p.c.pairs <= kMostFront;
  auto* kernel = kept ? append8_kernel<T, kHalves, true> : append8_kernel<T, kHalves, false>;
  return int(sm100::launch_overlapped(kernel, int((items * together + kWarps - 1) / kWarps), kThreads, 0, stream, p));
}

}  // namespace
}  // namespace latent

extern "C" int launch_latent_append8(void* stream, const latent_append8_call* call) {
  using namespace latent;
  if (call == nullptr) return -1;
  const latent_append_call& c = call->append;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || c.pairs < 8 || c.pairs > LATENT_MOST_PAIRS || c.pairs % 8 != 0) return -1;
  if (c.width < 2 * c.pairs || c.width % 16 != 0 || c.width > 65536) return -1;
  if (c.batches < 0 || c.batches > (1 << 26) || c.tokens < 0 || c.tokens > (int64_t(1) << 30) || c.pages < 0 || c.blocks < 0) return -1;
  if (c.page_rows < 64 || c.page_rows % 64 != 0 || c.pages > (INT32_MAX - 128) / c.page_rows || c.blocks > INT32_MAX / c.page_rows) return -1;
  if (call->block_rows < 1 || call->block_rows > 64 || (call->block_rows & (call->block_rows - 1)) != 0) return -1;
  if (!aligned(c.latent) || c.latent_token % 8 != 0 || !aligned(c.cache) || !fits_float(c.amplitude) || c.status == nullptr) return -1;
  if (c.tokens == 0 || c.batches == 0) return 0;
  Append8Params p = {c, call->scales, 0};
  while ((int64_t(1) << p.shift) < call->block_rows) ++p.shift;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c.type == LATENT_BF16) return c.layout ? launch_append8<__nv_bfloat16, true>(p, s) : launch_append8<__nv_bfloat16, false>(p, s);
  return c.layout ? launch_append8<__half, true>(p, s) : launch_append8<__half, false>(p, s);
}
