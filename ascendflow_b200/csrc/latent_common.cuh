// What the kernels around dense latent attention share: storage types, the turn of a pair of features, reports.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "../../include/latent.h"
#include "../../include/sparse_mla.h"
#include "tcgen05_ptx.cuh"

namespace latent {

__device__ __forceinline__ void report(int32_t* status, int code, int token, int detail) {
  if (atomicCAS(status, SPARSE_MLA_STATUS_OK, code) == SPARSE_MLA_STATUS_OK) {
    status[1] = token;
    status[2] = detail;
  }
}

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_float(float v) { return v; }

// Radians per position as a fraction of a turn, times 2^64: an angle is then a 64-bit product whose overflow is whole
// turns, exact for every position (the fraction is rounded once, to 53 bits). A frequency that is no number is none.
__device__ __forceinline__ uint64_t turns_of(double radians) {
  double turns = radians * 0.15915494309189533577;  // 1 / (2 pi)
  turns -= floor(turns);
  return turns >= 0.0 && turns < 1.0 ? uint64_t(turns * 18446744073709551616.0) : 0;
}
// (cos, sin) of `position` such fractions, times `amplitude`. The signed upper word is the angle in 2^-32 turns, within half a turn.
__device__ __forceinline__ float2 turn_of(int64_t position, uint64_t turns, float amplitude) {
  const int32_t fraction = int32_t((uint64_t(position) * turns + (uint64_t(1) << 31)) >> 32);
  float sine, cosine;
  sincospif(float(fraction) * 4.656612873077393e-10f, &sine, &cosine);  // 2^-31: half turns
  return make_float2(cosine * amplitude, sine * amplitude);
}

// A plain load, spelled out. (As `*at` it let the compiler arrange the expanded call's loop otherwise: 2K queries at 16K keys 314.0 us so, 316.1 with `*at`.)
__device__ __forceinline__ int fetch(const int32_t* at) {
  int value;
  asm volatile("ld.global.s32 %0, [%1];\n" : "=r"(value) : "l"(at));
  return value;
}
__device__ __forceinline__ int bounded(int value, int most) { return min(max(value, 0), most); }

// The request that owns `token` (binary search; empty requests are skipped), or -1 in front of the first and behind the last.
__device__ __forceinline__ int request_of(const int32_t* cu, int batches, int token) {
  if (token < *cu || token >= cu[batches]) return -1;
  int lo = 0, hi = batches;  // cu[lo] <= token < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= token) lo = mid; else hi = mid;
  }
  return lo;
}

// Finite in FP32, which the kernels work in.
inline bool fits_float(double value) { return value >= -FLT_MAX && value <= FLT_MAX; }
inline bool scale_fits(double value) { return value >= 1e-30 && value <= 1e30; }
inline bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline int multiprocessors() {
  static int cached[64] = {0};  // plain words written with the same value by whoever gets there first
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
  if (cached[device] == 0) {
    int count = 0;
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || count <= 0) count = 148;
    cached[device] = count;
  }
  return cached[device];
}

}  // namespace latent
