// What the attention kernels over latent rows use besides tcgen05_ptx.cuh: tensor copies into swizzled shared tiles, dense
// products of 128 rows, wide tensor-memory accesses.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcgen05_ptx.cuh"

namespace sm100 {

// ---- tensor copies ------------------------------------------------------------------------------------------------

// A box to shared memory; counts its bytes on `bar`. The first coordinate is a multiple of 16 bytes. What lies outside of the tensor is zero.
__device__ __forceinline__ void copy_box(uint32_t target, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n"
               ::"r"(target), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void copy_box(uint32_t target, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
               ::"r"(target), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// The map of a tensor of 16-bit values for boxes of 64 features (128 bytes, swizzled by 128) x `box_rows`. `sizes` from the innermost
// dimension outwards, `strides` (elements) of all but that; `row_dim` (1 or 2) is the dimension that the box's rows lie along.
// 0, or a CUDA error code.
inline int encode_map(CUtensorMap* map, int format, int rank, const void* base, const int64_t* sizes, const int64_t* strides, int row_dim, int box_rows) {
  using Encode = decltype(&cuTensorMapEncodeTiled);
  static Encode encode = nullptr;  // written with the same value by whoever gets there first
  if (encode == nullptr) {
    void* found = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (const cudaError_t error = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault, &result)) return int(error);
    if (result != cudaDriverEntryPointSuccess || found == nullptr) return int(cudaErrorNotSupported);
    encode = reinterpret_cast<Encode>(found);
  }
  cuuint64_t extent[3], bytes[2];
  cuuint32_t box[3] = {64, 1, 1}, steps[3] = {1, 1, 1};
  box[row_dim] = cuuint32_t(box_rows);
  for (int d = 0; d < rank; ++d) extent[d] = cuuint64_t(sizes[d]);
  for (int d = 0; d + 1 < rank; ++d) bytes[d] = cuuint64_t(strides[d]) * 2;
  const CUresult result = encode(map, format == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, cuuint32_t(rank), const_cast<void*>(base),
                                 extent, bytes, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return result == CUDA_SUCCESS ? 0 : int(cudaErrorInvalidValue);
}

// ---- dense products of 128 rows (one thread) -------------------------------------------------------------------------

template <bool kAccumulate>
__device__ __forceinline__ void mma_ss_c(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "n"(kAccumulate ? 1 : 0) : "memory");
}
// A from tensor memory: row i in lane i, two values to a column.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(uint32_t(accumulate)) : "memory");
}

// Limit (SM clocks, half a minute) of a wait that lasts as long as others work through many tiles; what they wait for by themselves has the usual one of a
// second, and whoever gives up ends all waits of the block.
constexpr long long kLongWait = 1ll << 36;

// For a role that has given up: waits (with the usual limit) for the products that this thread has issued, so that tensor memory can be given back.
__device__ __forceinline__ void wait_for_products(uint32_t unused_bar) {
  int never = 0;
  mma_commit(unused_bar);
  mbar_wait(unused_bar, 0, &never);
}

// ---- tensor memory -------------------------------------------------------------------------------------------------

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// 32 bytes (aligned) in one store: a whole sector of a lane's own row.
__device__ __forceinline__ void store_sector(void* at, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
               ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

__device__ __forceinline__ void load_sector(const void* at, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(at) : "memory");
}

// ---- arithmetic on pairs -------------------------------------------------------------------------------------------

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;\n" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;\n"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
// FP32 pair -> two words of the storage type (0: half, 1: bfloat16), rounded to nearest.
template <int kFormat>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kFormat == 1) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t&>(v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return reinterpret_cast<const uint32_t&>(v);
  }
}
__device__ __forceinline__ float greatest(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace sm100
