// Attention of bfloat16 queries over rows in 8 bits (included by latent_attention.cu): nothing of 16 bits goes through shared memory but the weights.
//
// Scores are products of 8-bit numbers. A query is split in two of them, q = 2^e (q1 + q2 / 16): four significant bits each make up bfloat16's eight, so what is
// left out is at most 2^-14 of 2^e, below 2^-21.8 of the row's greatest (448 2^e >= |q| > 224 2^e; e is not below -126, nor where the product with the scores' scale is no normal number). Lanes 0-15 of a subpartition hold q1 of 16 rows, lanes 16-31 q2, so that one product M = 128, N = 64 of 8 bits takes both; the
// softmax warps add the two sums and multiply by the key's scale and 2^e.
//
// The accumulator is turned: O^T = X^T P^T, features over the lanes and rows over the columns. X^T in 16 bits is the A operand, which the tensor core takes from tensor
// memory: a thread reads four features of 16 keys (a row's 128 bytes to a warp), widens them (latent_held8.cuh) and stores pairs of keys to its own lane. Lane l of
// subpartition s has features 4 (32 s + l) .. + 3, one in each of four products M = 128; which feature that is matters to the output only, where a thread then has
// four neighbours.
//
//   warps 0-3    softmax, rescaling, output
//   warps 4, 5   one thread each: S = Q X^T (8 bits); O^T += X^T P^T, 16 keys at a time
//   warp 6       chunks by tensor copies (boxes of 128 features x 64 rows, and one of 64) into a ring of five; the scales of their rows
//   warp 7       the plan
//   warps 8-15   Q of the next piece, split, to tensor memory (its last 64 features to shared memory)
//   warps 16-23  X^T, every other 16 keys by four of them, into two buffers in tensor memory
//
// What bounds it: the board's power (990 W) where a call is large. 64 requests of 64 heads at 32K, 1.22 GB: 379-385 us at 1.44 GHz, where the 16-bit products alone take 212 at the
// power limit's rate and reading at that rate as much energy as 155 us of it; 32 x 6 at 16K: 489-496 us at 1.63 GHz, 0.9 PFLOP/s. A chunk takes 2.3 k cycles: 18 products
// of 8 bits, 33 cycles each, 16 of 16 bits, and between those the chain of storing 16 widened keys to a buffer that has just become free. Against latent_held8.cuh
// (shared memory, 2.7 k cycles): 64 x 1 411 -> 379 us, 32 x 6 535 -> 489 on one board. Softmax by two groups of warps that take turns came down to 2.2 k cycles per chunk and
// took 388 and 508 us, since its instructions take power as well; waits that poll, or that are given a time, were slower.
//
// Tensor memory: columns 0-255 O^T (features' numbers modulo 4, 64 rows each), 256-383 Q's first 512 features, 384-447 scores, 448-511 X^T (two of 16 keys).
#pragma once

namespace latent {
namespace absorbed {
namespace turned {

constexpr int kQueryWarp0 = 8, kQueryWarps = 8, kConvertWarp0 = 16, kConvertWarps = 8, kThreads = 32 * (kConvertWarp0 + kConvertWarps);
constexpr int kRing = 5, kWideBoxBytes = kChunk * 128, kRestBoxBytes = kChunk * 64;
constexpr uint32_t kColumnsX = 448;
constexpr float kSecond = 16.f;  // q2 is held times this
constexpr int kLargeScale = 227, kSmallScale = 64, kBack = 20;

// What is said of a chunk's rows besides: factors of their scores (two halves, a bank apart), multipliers of their values for pairs of keys, and second ones.
struct Rows {
  float factors[2][kChunk / 2 + 4];
  uint32_t multipliers[kChunk / 2], again[kChunk / 2];
  int live, twice;
  float back;  // times this: 1 unless the scales are so large that sums of products times them do not fit FP32, or so small that they are subnormal, where the query's size may bring them back
  int pad;
};

template <int kWidth>
struct Layout {
  static constexpr int kTileBytes = kWidth * kChunk;
  static constexpr int kSmemP = kRing * kTileBytes;                       // two tiles of 64 rows x 64 weights
  static constexpr int kSmemRest = kSmemP + 2 * absorbed::kRows * 128;    // 128 lanes x 64 features of Q
  static constexpr int kSmemRows = kSmemRest + 128 * 64;                  // Rows[kRing]
  static constexpr int kSmemPieces = kSmemRows + kRing * int(sizeof(Rows));
  static constexpr int kSmemBars = kSmemPieces + kPieces * 64;
  static constexpr int kSmemAlpha = kSmemBars + 384;                      // float[2][64]
  static constexpr int kSmemInverse = kSmemAlpha + 2 * absorbed::kRows * 4;
  static constexpr int kSmemSize = kSmemInverse + absorbed::kRows * 4;    // float[2][64]: 2^e of the rows, of this piece and the next
  static constexpr int kSmemMost = kSmemSize + 2 * absorbed::kRows * 4;   // uint32[2][2][64]: rows' greatest magnitudes, by two warps each
  static constexpr int kSmemMisc = kSmemMost + 4 * absorbed::kRows * 4;
  static constexpr int kSmemBytes = kSmemMisc + 64 + 1024;
};
static_assert(Layout<576>::kSmemBytes <= 232448 && sizeof(Rows) % 16 == 0, "one block per SM");

// (the pieces' barriers are those of `Walk`)
enum Bar {
  kFull0 = absorbed::kPieceDone0 + kPieces, kFree0 = kFull0 + kRing, kQFull = kFree0 + kRing, kQFree, kScoresFull0, kScoresFree = kScoresFull0 + 2, kWeightsFull0, kWeightsFree0 = kWeightsFull0 + 2,
  kXFull0 = kWeightsFree0 + 2, kXFree0 = kXFull0 + 2, kMost0 = kXFree0 + 2, kSizes0 = kMost0 + 4, kMoved0 = kSizes0 + 2, kGivenUp0 = kMoved0 + 2, kGivenUp1, kBarCount
};
static_assert(kBarCount <= 48, "the barrier area");

__device__ __forceinline__ uint64_t smem_desc_sw64(uint32_t addr, uint32_t sbo) {
  return uint64_t((addr & 0x3FFFF) >> 4) | uint64_t(1) << 16 | uint64_t((sbo >> 4) & 0x3FFF) << 32 | uint64_t(1) << 46 | uint64_t(4) << 61;
}

// Products of 8-bit numbers with FP32 sums, A from tensor memory (row i in lane i, four values to a column) or shared memory.
template <bool kAccumulate>
__device__ __forceinline__ void mma8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "n"(kAccumulate ? 1 : 0) : "memory");
}
__device__ __forceinline__ void mma8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.eq.b32 p, 0, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ float2 multiply2(float2 a, float2 b) { return fma2(a, b, make_float2(0.f, 0.f)); }

inline int encode_map8(CUtensorMap* map, const void* base, int64_t width, int64_t rows, int box_features) {
  using Encode = decltype(&cuTensorMapEncodeTiled);
  static Encode encode = nullptr;  // written with the same value by whoever gets there first
  if (encode == nullptr) {
    void* found = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (const cudaError_t error = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault, &result)) return int(error);
    if (result != cudaDriverEntryPointSuccess || found == nullptr) return int(cudaErrorNotSupported);
    encode = reinterpret_cast<Encode>(found);
  }
  const cuuint64_t extent[2] = {cuuint64_t(width), cuuint64_t(rows)}, bytes[1] = {cuuint64_t(width)};
  const cuuint32_t box[2] = {cuuint32_t(box_features), kChunk}, steps[2] = {1, 1};
  const CUresult result = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), extent, bytes, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 box_features == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return result == CUDA_SUCCESS ? 0 : int(cudaErrorInvalidValue);
}

// ---- copies ---------------------------------------------------------------------------------------------------------

template <int kWidth>
__device__ __forceinline__ Rows* rows_of(const Shared& sm, uint32_t stage) { return reinterpret_cast<Rows*>(sm.ptr + Layout<kWidth>::kSmemRows) + stage; }

template <int kWidth>
__device__ void copy_role(const Params& p, const Shared& sm) {
  using L = Layout<kWidth>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0;
  bool given_up = false;
  Walk walk(sm);
  for (; !given_up && walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    if (piece.first == piece.last) continue;  // sees nothing
    const int32_t* table = p.table + size_t(piece.request) * p.pages;
    // Lane l: the first row of chunk `chunk + l` in the cache (below 2^31), or -1.
    auto first_row_of = [&](int chunk) {
      const int own = min(chunk + lane, piece.last - 1), column = over(own, p.by_page);
      const int page = column < p.pages ? table[column] : -1;
      return unsigned(page) < unsigned(p.blocks) ? page * p.page_rows + (own * kChunk - column * p.page_rows) : -1;
    };
    int rows = 0, next_rows = first_row_of(piece.first);  // of 32 chunks; of the next 32
    for (int chunk = piece.first; chunk < piece.last; ++chunk, ++count) {
      const int place = (chunk - piece.first) & 31;
      if (place == 0) {
        rows = next_rows;
        if (chunk + 32 < piece.last) next_rows = first_row_of(chunk + 32);
      }
      const int first = __shfl_sync(0xffffffffu, rows, place);
      const int valid = first >= 0 ? min(kChunk, piece.length - chunk * kChunk) : 0;
      int low = 0, high = 0;  // scales of rows 2 lane and 2 lane + 1
      if (first >= 0) {
        low = p.scales[(first + 2 * lane) >> p.block_shift];
        high = p.scales[(first + 2 * lane + 1) >> p.block_shift];
      }
      const uint32_t stage = count % kRing, use = count / kRing, target = sm.base + stage * L::kTileBytes, bar = sm.bar(kFull0 + stage);
      if (use > 0 && !warp_wait(sm.bar(kFree0 + stage), (use - 1) & 1, abort_flag)) { given_up = true; break; }
      Rows* about = rows_of<kWidth>(sm, stage);
      // What is behind the request's length, or in no page, has values of zero (as bits any byte is a finite number), and its scales count for nothing.
      const int most = __reduce_max_sync(0xffffffffu, max(low == 255 || 2 * lane >= valid ? 0 : low, high == 255 || 2 * lane + 1 >= valid ? 0 : high));
      const int up = most > kLargeScale ? -kBack : most < kSmallScale ? kBack : 0;
      // (what comes out as zero lies 60 binades below another scale of the chunk)
      auto factor_of = [&](int byte) { return __uint_as_float(byte == 255 ? 0x7fc00000u : uint32_t(max(byte + up, 0)) << 23); };
      *reinterpret_cast<float2*>(&about->factors[lane >> 4][2 * (lane & 15)]) = make_float2(factor_of(low), factor_of(high));
      const uint32_t first_one = 2 * lane < valid ? multiplier_of<1>(low) & 0xffffu : 0u, second_one = 2 * lane + 1 < valid ? multiplier_of<1>(high) << 16 : 0u;
      about->multipliers[lane] = first_one | second_one;
      about->again[lane] = (second_multiplier_of<1>(low) & 0xffffu) | second_multiplier_of<1>(high) << 16;
      if (lane == 0) {
        about->live = valid;
        about->twice = most > kMostInOne;
        about->back = __uint_as_float(uint32_t(127 - up) << 23);
        if (first < 0) report(p.status, SPARSE_MLA_STATUS_BAD_PAGE, int(piece.row / p.heads), chunk * kChunk);
      }
      __syncwarp();
      if (lane == 0) {
        if (first >= 0) {
          mbar_arrive_expect(bar, L::kTileBytes);
#pragma unroll
          for (int box = 0; box < 4; ++box) copy_box(target + box * kWideBoxBytes, &p.cache, box * 128, first, bar);
          if constexpr (kWidth == 576) copy_box(target + 4 * kWideBoxBytes, &p.rest, 512, first, bar);
        } else {
          mbar_arrive(bar);
        }
      }
      __syncwarp();
    }
  }
  if (*abort_flag != 0) {  // nothing of this block may be written behind its end
    int never = 0;
    for (uint32_t i = count > kRing ? count - kRing : 0; i < count; ++i) mbar_wait(sm.bar(kFull0 + i % kRing), (i / kRing) & 1, &never);
  }
}

// ---- queries --------------------------------------------------------------------------------------------------------

// Eight numbers, times `by`: q1 and q2 in two words each.
__device__ __forceinline__ void split8(const uint4& words, float by, uint2* one, uint2* two) {
  const uint32_t w[4] = {words.x, words.y, words.z, words.w};
  uint32_t first[4], second[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = __uint_as_float(w[e] << 16) * by, b = __uint_as_float(w[e] & 0xffff0000u) * by;
    uint16_t pair;
    uint32_t back;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(pair) : "f"(b), "f"(a));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(back) : "h"(pair));
    const float2 held = __half22float2(reinterpret_cast<const __half2&>(back));
    first[e] = pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(pair) : "f"((b - held.y) * kSecond), "f"((a - held.x) * kSecond));
    second[e] = pair;
  }
  *one = make_uint2(first[0] | first[1] << 16, first[2] | first[3] << 16);
  *two = make_uint2(second[0] | second[1] << 16, second[2] | second[3] << 16);
}

// As in the 16-bit form a subpartition's 16 rows are shared by two warps, segments of 64 bytes, a thread has 16 bytes of rows t / 4 and t / 4 + 8. The rows'
// greatest magnitudes first; then three segments at a time are read again (a loop: code that runs once per piece comes from far).
template <int kWidth>
__device__ void query_role(const Params& p, const Shared& sm, uint32_t tmem) {
  using L = Layout<kWidth>;
  const int warp = (threadIdx.x >> 5) - kQueryWarp0, lane = threadIdx.x & 31, subpartition = warp & 3, part = warp >> 2;
  volatile int* abort_flag = sm.abort_flag();
  constexpr int kOwn = kWidth / 64, kTogether = 3;  // segments of this warp; of them at a time
  const int row = subpartition * 16 + (lane >> 2), least = max(128 - int(__float_as_uint(p.scale_log2) >> 23), 1);
  uint32_t loads = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    if (piece.first == piece.last) continue;  // sees nothing
    const char* source = p.q + (piece.row + row) * (kWidth * 2) + (lane & 3) * 16;
    const int rows = piece.rows;
    auto fetch16 = [&](int s, int k) {
      const int segment = s < 8 ? part * 8 + s : 16 + part;
      uint4 words = make_uint4(0, 0, 0, 0);
      if (row + 8 * k < rows && s < kOwn) words = *reinterpret_cast<const uint4*>(source + k * 8 * (kWidth * 2) + segment * 64);
      return words;
    };
    uint32_t greatest[2] = {0, 0};
#pragma unroll 1
    for (int s0 = 0; s0 < kOwn; s0 += 5) {
      uint4 words[5][2];
#pragma unroll
      for (int s = 0; s < 5; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) words[s][k] = fetch16(s0 + s, k);
#pragma unroll
      for (int s = 0; s < 5; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (const uint32_t w : {words[s][k].x, words[s][k].y, words[s][k].z, words[s][k].w})
            greatest[k] = max(greatest[k], max(w & 0x7fffu, w >> 16 & 0x7fffu));  // (bits of bfloat16 numbers grow with them)
    }
    uint32_t* most = reinterpret_cast<uint32_t*>(sm.ptr + L::kSmemMost);
    float* sizes = reinterpret_cast<float*>(sm.ptr + L::kSmemSize);
    const uint32_t parity = loads & 1;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      greatest[k] = max(greatest[k], __shfl_xor_sync(0xffffffffu, greatest[k], 1));
      greatest[k] = max(greatest[k], __shfl_xor_sync(0xffffffffu, greatest[k], 2));
      if ((lane & 3) == 0) most[(parity * 2 + part) * kRows + row + 8 * k] = greatest[k];
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.bar(kMost0 + subpartition));
    uint4 words[kTogether][2];
#pragma unroll
    for (int s = 0; s < kTogether; ++s)
#pragma unroll
      for (int k = 0; k < 2; ++k) words[s][k] = fetch16(s, k);
    if (!warp_wait(sm.bar(kMost0 + subpartition), parity, abort_flag, kLongWait)) return;
    float by[2], size[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t bits = max(greatest[k], most[(parity * 2 + (part ^ 1)) * kRows + row + 8 * k]) << 16;
      // 2^e: the least with |q| <= 448 2^e, a normal number as its inverse is, and the product with the scores' scale (rows of zeros, tiny ones: what is left out of these moves scores by less
      // than 2^-138 of the keys' magnitudes). A row with what is no number, or infinite, has none: all of its scores are NaN, and only those of keys that it sees are taken.
      const int e = min(max(int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u), least), 253);
      by[k] = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(uint32_t(254 - e) << 23);
      size[k] = __uint_as_float(uint32_t(e) << 23);
    }
    if (loads > 0 && !warp_wait(sm.bar(kQFree), (loads - 1) & 1, abort_flag, kLongWait)) return;
    tc_fence_after_sync();
    // (the products of the piece in front have ended, so the softmax warps have the sizes of the one in front of that)
    if (part == 0) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if ((lane & 3) == 0) sizes[parity * kRows + row + 8 * k] = size[k];
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kSizes0 + parity));
    }
#pragma unroll 1
    for (int s0 = 0; s0 < kOwn; s0 += kTogether) {
      uint4 next[kTogether][2];
#pragma unroll
      for (int s = 0; s < kTogether; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) next[s][k] = fetch16(s0 + kTogether + s, k);
#pragma unroll
      for (int s = 0; s < kTogether; ++s) {
        uint2 a1, a2, b1, b2;
        split8(words[s][0], by[0], &a1, &a2);
        split8(words[s][1], by[1], &b1, &b2);
        if (s0 + s < 8) {
          const uint32_t at = tmem + (uint32_t(subpartition * 32) << 16) + kColumnsQ + (part * 8 + s0 + s) * 8;
          tmem_st_8(at, a1.x, a1.y, b1.x, b1.y);
          tmem_st_8(at + kHighLanes, a2.x, a2.y, b2.x, b2.y);
        } else if (kOwn > 8 && s0 + s == 8) {  // rows of 64 bytes, swizzled by 64
          auto place = [&](int lane_of) {
            return reinterpret_cast<uint2*>(sm.ptr + L::kSmemRest + lane_of * 64 + (((part * 2 + ((lane & 3) >> 1)) ^ (lane_of >> 1 & 3)) << 4) + (lane & 1) * 8);
          };
          const int low = subpartition * 32 + (lane >> 2);
          *place(low) = a1;
          *place(low + 8) = b1;
          *place(low + 16) = a2;
          *place(low + 24) = b2;
        }
      }
#pragma unroll
      for (int s = 0; s < kTogether; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) words[s][k] = next[s][k];
    }
    tmem_wait_st();
    fence_proxy_async();  // products read the last features through the async proxy
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.bar(kQFull));
    ++loads;
  }
}

// ---- values ---------------------------------------------------------------------------------------------------------

// Byte kByte of `a` and of `b`, times `factors`.
template <int kByte>
__device__ __forceinline__ uint32_t widened_pair(uint32_t a, uint32_t b, uint32_t factors) {
  uint32_t spread;
  asm("prmt.b32 %0, %1, %2, %3;\n" : "=r"(spread) : "r"(a), "r"(b), "n"(0xc480 + 0x1111 * kByte));
  return multiply_pair<1>(spread << 4 & 0x87f087f0u, factors);
}

template <int kWidth>
__device__ void convert_role(const Shared& sm, uint32_t tmem) {
  using L = Layout<kWidth>;
  const int warp = (threadIdx.x >> 5) - kConvertWarp0, lane = threadIdx.x & 31, subpartition = warp & 3, buffer = warp >> 2;
  volatile int* abort_flag = sm.abort_flag();
  const uint32_t target = tmem + (uint32_t(subpartition * 32) << 16) + kColumnsX + buffer * 32;
  // Four features of a key: the swizzle exchanges a row's units of 16 bytes by its number.
  const uint32_t source = sm.base + subpartition * kWideBoxBytes + ((lane >> 2) << 4) + (lane & 3) * 4;
  uint32_t count = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    for (int left = walk.piece.last - walk.piece.first; left > 0; --left, ++count) {
      const uint32_t stage = count % kRing;
      if (!warp_wait(sm.bar(kFull0 + stage), (count / kRing) & 1, abort_flag)) return;
      const Rows* about = rows_of<kWidth>(sm, stage);
      const bool twice = about->twice != 0;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int group = 2 * half + buffer;  // of 16 keys
        const uint32_t number = 2 * count + half, from = source + stage * L::kTileBytes + group * 16 * 128;
        uint32_t raw[16], factors[8];
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(raw[i]) : "r"((from ^ ((i & 7) << 4)) + i * 128) : "memory");
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(&about->multipliers[group * 8 + i]);
          factors[i] = v.x;
          factors[i + 1] = v.y;
          factors[i + 2] = v.z;
          factors[i + 3] = v.w;
        }
        uint32_t words[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          words[i] = widened_pair<0>(raw[2 * i], raw[2 * i + 1], factors[i]);
          words[8 + i] = widened_pair<1>(raw[2 * i], raw[2 * i + 1], factors[i]);
          words[16 + i] = widened_pair<2>(raw[2 * i], raw[2 * i + 1], factors[i]);
          words[24 + i] = widened_pair<3>(raw[2 * i], raw[2 * i + 1], factors[i]);
        }
        if (twice) {  // (scales above 2^7)
#pragma unroll
          for (int i = 0; i < 32; ++i) words[i] = multiply_pair<1>(words[i], about->again[group * 8 + (i & 7)]);
        }
        // (everything is ready before the buffer is free: what the products wait for is short)
        if (number > 0 && !warp_wait(sm.bar(kXFree0 + buffer), (number - 1) & 1, abort_flag)) return;
        tc_fence_after_sync();
        tmem_st32(target, words);
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(kXFull0 + buffer));
      }
      if (lane == 0) mbar_arrive(sm.bar(kFree0 + stage));
    }
  }
}

// ---- products (one thread each) --------------------------------------------------------------------------------------

constexpr uint32_t kIdescScores = idesc_f16(128, kChunk, 0, 0, 0);  // (format 0: e4m3 where the kind is of 8 bits)
constexpr uint32_t kIdescValues = idesc_f16(128, kRows, 1, 0, 0);

template <int K = 0>
__device__ __forceinline__ void issue_scores(uint32_t tmem, uint64_t x_desc) {
  if constexpr (K < 16) {
    mma8_ts<K != 0>(tmem + kColumnsScores, tmem + kColumnsQ + K * 8, x_desc + (((K >> 2) * kWideBoxBytes + (K & 3) * 32) >> 4), kIdescScores);
    issue_scores<K + 1>(tmem, x_desc);
  }
}

template <int kWidth>
__device__ void score_role(const Shared& sm, uint32_t tmem) {
  using L = Layout<kWidth>;
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0, loads = 0;
  Walk walk(sm);
  const uint64_t q_rest = smem_desc_sw64(sm.base + L::kSmemRest, 512);
  for (; walk.next_of_thread(); walk.done()) {
    const int chunks = walk.piece.last - walk.piece.first;
    if (chunks == 0) continue;
    if (!mbar_wait(sm.bar(kQFull), loads++ & 1, abort_flag)) return;
    for (int i = 0; i < chunks; ++i, ++count) {
      const uint32_t stage = count % kRing, tile = sm.base + stage * L::kTileBytes;
      if (!mbar_wait(sm.bar(kFull0 + stage), (count / kRing) & 1, abort_flag)) return;
      if (!mbar_wait(sm.bar(kScoresFree), (count & 1) ^ 1, abort_flag)) return;
      tc_fence_after_sync();
      issue_scores(tmem, smem_desc_sw128(tile, 16, 1024));
      if constexpr (kWidth == 576) {
        const uint64_t x_rest = smem_desc_sw64(tile + 4 * kWideBoxBytes, 512);
        mma8_ss(tmem + kColumnsScores, q_rest, x_rest, kIdescScores);
        mma8_ss(tmem + kColumnsScores, q_rest + 2, x_rest + 2, kIdescScores);
      }
      mma_commit(sm.bar(kScoresFull0 + (count & 1)));
      mma_commit(sm.bar(kFree0 + stage));
    }
    mma_commit(sm.bar(kQFree));
  }
}

template <int kWidth>
__device__ void value_role(const Shared& sm, uint32_t tmem) {
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0;
  Walk walk(sm);
  const uint64_t p_desc = smem_desc_sw128(sm.base + Layout<kWidth>::kSmemP, 16, 1024);
  // The scores of a chunk are said to be there when the products of the chunk before the last have ended, too: one wait for both. (The first two have no such chunk.)
  mbar_arrive(sm.bar(kScoresFull0));
  mbar_arrive(sm.bar(kScoresFull0 + 1));
  for (; walk.next_of_thread(); walk.done()) {
    const int chunks = walk.piece.last - walk.piece.first;
    for (int i = 0; i < chunks; ++i, ++count) {
      const uint32_t tile = count & 1;
      if (!mbar_wait(sm.bar(kWeightsFull0 + tile), (count >> 1) & 1, abort_flag)) return;
#pragma unroll
      for (int group = 0; group < 4; ++group) {
        const uint32_t number = 2 * count + group / 2;
        if (!mbar_wait(sm.bar(kXFull0 + (group & 1)), number & 1, abort_flag)) return;
        tc_fence_after_sync();
#pragma unroll
        for (int m = 0; m < 4; ++m)
          mma_ts(tmem + m * kRows, tmem + kColumnsX + (group & 1) * 32 + m * 8, p_desc + ((tile * kRows * 128 + group * 32) >> 4), kIdescValues, i > 0 || group > 0);
        mma_commit(sm.bar(kXFree0 + (group & 1)));
      }
      mma_commit(sm.bar(kWeightsFree0 + tile));
      mma_commit(sm.bar(kScoresFull0 + tile));
    }
  }
}

// ---- softmax ----------------------------------------------------------------------------------------------------------

// References and sums as in the 16-bit form's `softmax_role`; weights go to two tiles in turn, the accumulator's columns are rows.
template <int kWidth>
__device__ void softmax_role(const Params& p, const Shared& sm, uint32_t tmem) {
  using L = Layout<kWidth>;
  constexpr int kFormat = 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4;
  volatile int* abort_flag = sm.abort_flag();
  const uint32_t lanes = uint32_t(warp * 32) << 16, scores = tmem + kColumnsScores + lanes;
  const int row = warp * 16 + (lane & 15), feature = 4 * (warp * 32 + lane);
  float* alphas = reinterpret_cast<float*>(sm.ptr + L::kSmemAlpha);
  float* inverses = reinterpret_cast<float*>(sm.ptr + L::kSmemInverse);
  const float* sizes = reinterpret_cast<const float*>(sm.ptr + L::kSmemSize);
  int* moved = reinterpret_cast<int*>(sm.ptr + L::kSmemMisc + 16);  // [2][4]
  // The four warps meet at outputs. One whose wait gave up says so there, and all leave behind it.
  bool failed = false;
  constexpr uint32_t kGivenUp = 32;
  auto meet = [&](bool flag) { return named_barrier_count(1, 32 * kSoftmaxWarps, failed || (flag && lane == 0)); };
  // The end of the products of chunk `index`.
  auto products_end = [&](uint32_t index) { return warp_wait(sm.bar(kWeightsFree0 + (index & 1)), (index >> 1) & 1, abort_flag); };
  uint32_t count = 0, loads = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    const int chunks = piece.last - piece.first;
    const int end = row < piece.rows ? piece.base + over(piece.head + row, p.by_heads) + piece.token : INT32_MAX;  // this row sees keys below
    const int warp_end = __reduce_min_sync(0xffffffffu, end);
    float reference = -INFINITY, sum = 0.f, scale = 0.f;
    if (chunks > 0) {
      if (!warp_wait(sm.bar(kSizes0 + (loads & 1)), (loads >> 1) & 1, abort_flag, kLongWait)) { failed = true; meet(true); return; }
      scale = fminf(p.scale_log2 * sizes[(loads++ & 1) * kRows + row], FLT_MAX);
    }
    for (int i = 0; i < chunks; ++i, ++count) {
      const uint32_t stage = count % kRing;
      // (the tile has landed when its scores are there; this wait makes what was written about it visible)
      if (!warp_wait(sm.bar(kScoresFull0 + (count & 1)), (count >> 1) & 1, abort_flag) || !warp_wait(sm.bar(kFull0 + stage), (count / kRing) & 1, abort_flag)) { failed = true; meet(true); return; }
      tc_fence_after_sync();
      const Rows* about = rows_of<kWidth>(sm, stage);
      const int key = (piece.first + i) * kChunk, live = about->live;
      // (a positive number, for masked scores and zeros are multiplied by it, too; what the bounds move are scores below 2^-140, or beyond FP32)
      const float scale_log2 = fminf(fmaxf(scale * about->back, FLT_MIN), FLT_MAX);
      float2 s[16];
      {
        uint32_t low_a[16], low_b[16], high_a[16], high_b[16];
        tmem_ld16_halves<32>(scores, low_a);
        tmem_ld16_halves<32>(scores + 16, low_b);
        tmem_ld16_halves<32>(scores + kHighLanes, high_a);
        tmem_ld16_halves<32>(scores + kHighLanes + 16, high_b);
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(kScoresFree));
        const float2 part = make_float2(1.f / kSecond, 1.f / kSecond);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[e] = fma2(make_float2(__uint_as_float(high_a[2 * e]), __uint_as_float(high_a[2 * e + 1])), part, make_float2(__uint_as_float(low_a[2 * e]), __uint_as_float(low_a[2 * e + 1])));
          s[8 + e] = fma2(make_float2(__uint_as_float(high_b[2 * e]), __uint_as_float(high_b[2 * e + 1])), part,
                          make_float2(__uint_as_float(low_b[2 * e]), __uint_as_float(low_b[2 * e + 1])));
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float4 f = *reinterpret_cast<const float4*>(&about->factors[half][2 * e]);
        s[e] = multiply2(s[e], make_float2(f.x, f.y));
        s[e + 1] = multiply2(s[e + 1], make_float2(f.z, f.w));
      }
      if (live < kChunk || key + kChunk > warp_end) {
        const int seen = min(end - key, live) - half * 32;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (2 * e >= seen) s[e].x = -INFINITY;
          if (2 * e + 1 >= seen) s[e].y = -INFINITY;
        }
      }
      float most[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        most[k] = fmaxf(s[4 * k].x, s[4 * k].y);
#pragma unroll
        for (int e = 1; e < 4; ++e) most[k] = greatest(most[k], s[4 * k + e].x, s[4 * k + e].y);
      }
      const float own = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * scale_log2;  // scale > 0
      const bool look = __any_sync(0xffffffffu, own > reference + kRoom);
      float alpha = 1.f;
      if (look) {
        const float top = fmaxf(own, __shfl_xor_sync(0xffffffffu, own, 16));
        if (top > reference + kRoom) {
          const float next = top - (reference == -INFINITY ? kFirst<kFormat> : kStep);
          alpha = exp2f(reference - next);
          reference = next;
        }
      }
      // Who has moved a reference is told here, and asked when the weights are there.
      float* factors = alphas + (count & 1) * kRows;
      if (half == 0) factors[row] = alpha;
      if (lane == 0) moved[(count & 1) * kSoftmaxWarps + warp] = look && i > 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kMoved0 + (count & 1)));
      const float shift = reference == -INFINITY ? 0.f : -reference;
      const float2 scales = make_float2(scale_log2, scale_log2), shifts = make_float2(shift, shift);
      float2 sum_a = make_float2(0.f, 0.f), sum_b = sum_a;
      uint4 packed[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t words[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int e = 4 * u + w;
          float2 weight = fma2(s[e], scales, shifts);
          weight.x = exp2f(weight.x);
          weight.y = exp2f(weight.y);
          if (e & 1) sum_b = add2(sum_b, weight); else sum_a = add2(sum_a, weight);
          words[w] = pack2<kFormat>(weight.x, weight.y);
        }
        packed[u] = make_uint4(words[0], words[1], words[2], words[3]);
      }
      sum = sum * alpha + ((sum_a.x + sum_a.y) + (sum_b.x + sum_b.y));
      unsigned char* weights = sm.ptr + L::kSmemP + (count & 1) * kRows * 128;
#pragma unroll
      for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4*>(weights + row * 128 + (((half * 4 + u) ^ (row & 7)) << 4)) = packed[u];
      if (!warp_wait(sm.bar(kMoved0 + (count & 1)), (count >> 1) & 1, abort_flag)) { failed = true; meet(true); return; }
      const int4 any = *reinterpret_cast<const int4*>(moved + (count & 1) * kSoftmaxWarps);
      if ((any.x | any.y | any.z | any.w) != 0) {
        if (!products_end(count - 1)) { failed = true; meet(true); return; }
        tc_fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < 256; c += 32) {
          uint32_t o[32];
          tmem_ld32(tmem + c + lanes, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 by = *reinterpret_cast<const float4*>(factors + (c & 63) + e);
            o[e] = __float_as_uint(__uint_as_float(o[e]) * by.x);
            o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) * by.y);
            o[e + 2] = __float_as_uint(__uint_as_float(o[e + 2]) * by.z);
            o[e + 3] = __float_as_uint(__uint_as_float(o[e + 3]) * by.w);
          }
          tmem_st32(tmem + c + lanes, o);
        }
        tmem_wait_st();
      }
      fence_proxy_async();  // the product reads the weights through the async proxy
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kWeightsFull0 + (count & 1)));
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    // ---- output
    if (chunks > 0) {
      if (!products_end(count - 1)) { failed = true; meet(true); return; }
      tc_fence_after_sync();
    }
    if (piece.slot >= 0) {  // a part of a tile: sums as they are
      if (half == 0 && row < piece.rows) p.statistics[size_t(piece.slot) * kRows + row] = part_statistics(reference, sum);
    } else {
      float log_sum;
      const float sink = p.sinks != nullptr && row < piece.rows ? p.sinks[(piece.head + row) % p.heads] * kLog2E : -INFINITY;
      const float inverse = inverse_of(reference, sum, sink, &log_sum);
      if (half == 0) {
        inverses[row] = inverse;
        if (p.lse != nullptr && row < piece.rows) p.lse[piece.row + row] = log_sum * kLn2;
      }
      if (meet(false) != 0) return;
    }
    float* sums = p.sums + size_t(max(piece.slot, 0)) * kSlotFloats + feature;
    char* out = p.out + (piece.row * LATENT_VALUES + feature) * 2;
#pragma unroll 1
    for (int first = 0; first < piece.rows; first += 8) {
      uint32_t o[4][8];
      if (chunks > 0) {
#pragma unroll
        for (int m = 0; m < 4; ++m) tmem_ld8(tmem + lanes + m * kRows + first, o[m]);
        tmem_wait_ld();
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (first + e >= piece.rows) break;
        if (piece.slot >= 0) {
          *reinterpret_cast<uint4*>(sums + (first + e) * LATENT_VALUES) = make_uint4(o[0][e], o[1][e], o[2][e], o[3][e]);
        } else {
          const float by = inverses[first + e];
          uint2 words = make_uint2(0, 0);
          if (chunks > 0 && by != 0.f)
            words = make_uint2(pack2<kFormat>(__uint_as_float(o[0][e]) * by, __uint_as_float(o[1][e]) * by), pack2<kFormat>(__uint_as_float(o[2][e]) * by, __uint_as_float(o[3][e]) * by));
          *reinterpret_cast<uint2*>(out + (first + e) * (LATENT_VALUES * 2)) = words;
        }
      }
    }
    if (piece.slot < 0 && meet(false) != 0) return;  // the inverses are free again
  }
  if (*abort_flag != 0) failed = true;
  meet(false);  // with a warp that has given up since the last time
}

// ---- kernel -----------------------------------------------------------------------------------------------------------

// Registers: 128 for a softmax thread, 56 for the warps that issue, copy and plan, 72 for the others, of 6 x 80.
template <int kWidth>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ Params p) {
  using L = Layout<kWidth>;
  extern __shared__ unsigned char smem_raw[];
  Shared sm;
  const uint32_t raw = smem_u32(smem_raw), pad = (1024u - (raw & 1023u)) & 1023u;
  sm.base = raw + pad;
  sm.ptr = smem_raw + pad;
  sm.bars = L::kSmemBars;
  sm.pieces = L::kSmemPieces;
  sm.misc = L::kSmemMisc;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarCount; ++i) {
      int arrivals = 1;
      if (i >= kFree0 && i < kFree0 + kRing) arrivals = 1 + kConvertWarps;
      else if (i >= kPieceDone0 && i < kPieceDone0 + kPieces) arrivals = kSoftmaxWarps + 3 + kQueryWarps + kConvertWarps;
      else if (i == kQFull) arrivals = kQueryWarps;
      else if (i == kScoresFree || (i >= kWeightsFull0 && i < kWeightsFull0 + 2) || (i >= kMoved0 && i < kMoved0 + 2)) arrivals = kSoftmaxWarps;
      else if (i >= kScoresFull0 && i < kScoresFull0 + 2) arrivals = 2;
      else if (i >= kXFull0 && i < kXFull0 + 2) arrivals = kConvertWarps / 2;
      else if (i >= kMost0 && i < kMost0 + 4) arrivals = 2;
      else if (i >= kSizes0 && i < kSizes0 + 2) arrivals = kQueryWarps / 2;
      mbar_init(sm.bar(i), arrivals);
    }
    mbar_fence_init();
    *sm.abort_flag() = 0;
  }
  if (warp == kScoreWarp) { tmem_alloc(smem_u32(sm.tmem_slot()), 512); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *sm.tmem_slot();
  wait_for_predecessor();
  let_successor_start();
  Place place = {};
  Borders borders = {};
  if (p.batches > 32) {
    borders = plan_block<kThreads / 32>(p, sm.scan(), &place);
    fence_proxy_async();  // the plan's scratch is the first tile's memory
    __syncthreads();
  }
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;\n");
    turned::softmax_role<kWidth>(p, sm, tmem);
  } else if (warp < kQueryWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
    if (warp == kScoreWarp || warp == kValueWarp) {
      if (elect_one()) {
        if (warp == kScoreWarp) turned::score_role<kWidth>(sm, tmem);
        else turned::value_role<kWidth>(sm, tmem);
        if (*sm.abort_flag() != 0) wait_for_products(sm.bar(warp == kScoreWarp ? kGivenUp0 : kGivenUp1));
      }
      __syncwarp();
    } else if (warp == kCopyWarp) {
      turned::copy_role<kWidth>(p, sm);
    } else {
      if (p.batches <= 32) borders = plan_block<1>(p, nullptr, &place);
      plan_role(p, sm, borders, place);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
    if (warp < kConvertWarp0) turned::query_role<kWidth>(p, sm, tmem);
    else turned::convert_role<kWidth>(sm, tmem);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && *sm.abort_flag() != 0) report(p.status, SPARSE_MLA_STATUS_WAIT_EXPIRED, blockIdx.x, 0);
  if (warp == kScoreWarp) tmem_dealloc(tmem, 512);
}

}  // namespace turned
}  // namespace absorbed
}  // namespace latent
