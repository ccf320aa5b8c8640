// Attention over a long axis by several blocks: each leaves unnormalised sums of its part in FP32, with a reference (log2) and a sum of weights per row;
// here they are added up.
//
// sum = sum_i 2^(reference_i - reference) sum_i, and the same for the rows' features; a part in which a row sees nothing has reference -infinity, sum 0.
#pragma once

#include "latent_ptx.cuh"

namespace latent {

using namespace sm100;

constexpr int kUnitRows = 8, kUnitFeatures = 32, kPartsInFlight = 4;
constexpr int kCombineThreads = 256, kCombineWarps = kCombineThreads / 32;

struct alignas(16) Shares {  // what the warps of a block have; read and written 16 bytes at a time
  float sums[kCombineWarps][kUnitRows * kUnitFeatures];
  float2 statistics[kCombineWarps][kUnitRows];
};

// (a row whose scores are NaNs has no greatest one, but its sum is to be a NaN)
__device__ __forceinline__ float2 part_statistics(float reference, float sum) { return make_float2(reference == -INFINITY && sum != 0.f ? 0.f : reference, sum); }

// Warps that work on eight rows x 32 features: as many as bring all parts with one round of loads.
__device__ __forceinline__ int warps_for(int parts) {
  return parts <= kPartsInFlight ? 1 : parts <= 2 * kPartsInFlight ? 2 : parts <= 4 * kPartsInFlight ? 4 : kCombineWarps;
}

// Rows `rows` .. + 7 (those below `limit`), 32 features of them, by `warps` (a power of two, the same for the whole block) neighbouring warps; every
// `warps`-th part is one's. Lane l adds up eight features of row l % 8: sums_of(part, row) and statistics_of(part, row) are where this lane's lie,
// place_of(row, lane) where those of `lane` go, finish(row, reference, sum, is it the row's first feature) what they are multiplied with.
template <int kFormat, class SumsOf, class StatisticsOf, class PlaceOf, class Finish>
__device__ __forceinline__ void join_parts(Shares& shares, int warps, int parts, int rows, int limit, SumsOf sums_of, StatisticsOf statistics_of, PlaceOf place_of, Finish finish) {
  static_assert(kPartsInFlight == 4, "a part for every eight lanes");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = warp & (warps - 1);
  const int row = rows + (lane & 7), count = (parts - first + warps - 1) / warps;
  float total[8] = {}, reference = -INFINITY, sum = 0.f;
  for (int round = 0; round < count; round += kPartsInFlight) {
    uint32_t v[kPartsInFlight][8];
#pragma unroll
    for (int n = 0; n < kPartsInFlight; ++n)
      if (round + n < count) load_sector(sums_of(first + (round + n) * warps, row), v[n]);
    const int mine = round + (lane >> 3);  // lane l has the statistics of part l / 8 of the round
    const float2 own = mine < count ? *statistics_of(first + mine * warps, row) : make_float2(-INFINITY, 0.f);
    float next = fmaxf(reference, own.x);
    next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 8));
    next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 16));
    const float factor = own.x == -INFINITY ? 0.f : exp2f(own.x - next);
    float more = factor * own.y;
    more += __shfl_xor_sync(0xffffffffu, more, 8);
    more += __shfl_xor_sync(0xffffffffu, more, 16);
    const float alpha = reference == -INFINITY ? 0.f : exp2f(reference - next);
    sum = sum * alpha + more;
    reference = next;
#pragma unroll
    for (int e = 0; e < 8; ++e) total[e] *= alpha;
#pragma unroll
    for (int n = 0; n < kPartsInFlight; ++n) {
      if (round + n >= count) break;
      const float by = __shfl_sync(0xffffffffu, factor, n * 8 + (lane & 7));
      if (by != 0.f) {  // (what a part in which the row sees nothing has there may be anything)
#pragma unroll
        for (int e = 0; e < 8; ++e) total[e] += __uint_as_float(v[n][e]) * by;
      }
    }
  }
  if (warps == 1) {  // (no barrier in this branch)
    if (row < limit) {
      const float inverse = finish(row, reference, sum, lane < 8);
      uint32_t words[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) words[e] = inverse == 0.f ? 0u : pack2<kFormat>(total[2 * e] * inverse, total[2 * e + 1] * inverse);
      *reinterpret_cast<uint4*>(place_of(row, lane)) = make_uint4(words[0], words[1], words[2], words[3]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(&shares.sums[warp][lane * 8 + e]) = make_float4(total[e], total[e + 1], total[e + 2], total[e + 3]);
  if (lane < 8) shares.statistics[warp][lane] = make_float2(reference, sum);
  __syncthreads();
  for (int pair = first * 32 + lane; pair < kUnitRows * kUnitFeatures / 2; pair += warps * 32) {
    const int owner = pair >> 2, row = rows + (owner & 7);  // the lane that had it
    if (row >= limit) continue;
    float reference = -INFINITY, sum = 0.f;
    for (int w = 0; w < warps; ++w) reference = fmaxf(reference, shares.statistics[warp - first + w][owner & 7].x);
    float2 value = make_float2(0.f, 0.f);
    for (int w = 0; w < warps; ++w) {
      const float2 share = *reinterpret_cast<const float2*>(&shares.sums[warp - first + w][pair * 2]), own = shares.statistics[warp - first + w][owner & 7];
      const float by = own.x == -INFINITY ? 0.f : exp2f(own.x - reference);
      value.x += share.x * by;
      value.y += share.y * by;
      sum += own.y * by;
    }
    const float inverse = finish(row, reference, sum, pair < 32 && (pair & 3) == 0);
    *reinterpret_cast<uint32_t*>(place_of(row, owner) + (pair & 3) * 4) = inverse == 0.f ? 0u : pack2<kFormat>(value.x * inverse, value.y * inverse);
  }
  __syncthreads();  // the shares may be overwritten
}

}  // namespace latent
