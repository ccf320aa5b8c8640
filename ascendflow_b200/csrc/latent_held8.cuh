// Rows held in 8 bits on their way into the absorbed attention kernel's tiles (included by latent_attention.cu).
//
// A value is an e4m3 number times its block's scale, a power of two: in 16 bits the product is exact, so products, softmax and sums are those
// of a 16-bit cache that holds the same numbers. Of s.eeee.mmm the bits moved to s.0000eeee.mmm0000 are, as bfloat16, the value times
// 2^-120 (subnormal numbers too), and to s.0eeee.mmm0000000, as half, times 2^-8; one multiplication of a pair by the scale times 2^120 or 2^8 does the
// rest: a permutation, a shift, a mask and a product for two values.
//
//   warps 8-11   Q of the next piece from global to tensor memory (a subpartition each)
//   warps 12-19  chunks: 64 rows of W bytes, nine (eight) loads of 16 bytes per thread, sixteen values to 32 bytes of the tile each. What is loaded
//                for the next chunk takes the place of what has been stored, so that loads are always on their way.
#pragma once

namespace latent {
namespace absorbed {

constexpr int kQueryWarps8 = 4, kConvertWarp0 = kQueryWarp0 + kQueryWarps8, kConvertWarps = 8;
constexpr int kThreads8 = 32 * (kConvertWarp0 + kConvertWarps);

// A scale's byte: 2^(byte - 127), 255: NaN. The multiplier (twice, for a pair) is 2^(byte - kBias); what is above the type's largest power of two is
// left for a second one.
template <int kFormat> constexpr int kBias = kFormat == 1 ? 7 : 119;
constexpr int kMostInOne = 134;  // 2^127 in bfloat16, 2^15 in half
template <int kFormat>
__device__ __forceinline__ uint32_t power_of_two(int exponent) {  // (below the type's range: zero)
  uint32_t bits;
  if constexpr (kFormat == 1) bits = uint32_t(exponent + 127) << 7;
  else bits = exponent >= -14 ? uint32_t(exponent + 15) << 10 : exponent >= -24 ? 1u << (exponent + 24) : 0u;
  return bits | bits << 16;
}
template <int kFormat>
__device__ __forceinline__ uint32_t multiplier_of(int byte) {
  if (byte == 255) return 0x7fff7fffu;  // NaN in either type
  return power_of_two<kFormat>(min(byte, kMostInOne) - kBias<kFormat>);
}
// (half: values times such scales are finite up to 2^22 only, where this is 2^15)
template <int kFormat>
__device__ __forceinline__ uint32_t second_multiplier_of(int byte) {
  const int rest = byte == 255 ? 0 : max(byte - kMostInOne, 0);
  return power_of_two<kFormat>(kFormat == 1 ? rest : min(rest, 15));
}

template <int kFormat>
__device__ __forceinline__ uint32_t multiply_pair(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (kFormat == 1) asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  else asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Bytes 2 kHalf and 2 kHalf + 1 of `word`, times `factor`. (The permutation puts a byte's sign over eight bits, of which the mask leaves the highest.)
template <int kFormat, int kHalf>
__device__ __forceinline__ uint32_t widened(uint32_t word, uint32_t factor) {
  uint32_t spread;
  asm("prmt.b32 %0, %1, 0, %2;\n" : "=r"(spread) : "r"(word), "n"(kHalf ? 0xb3a2 : 0x9180));
  return multiply_pair<kFormat>(kFormat == 1 ? spread << 4 & 0x87f087f0u : spread << 7 & 0xbf80bf80u, factor);
}

__device__ __forceinline__ uint4 load_held(const char* at) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at) : "memory");
  return v;
}

template <int kFormat, int kWidth>
__device__ void convert_role(const Params& p, const Shared& sm) {
  using L = Layout<kWidth>;
  constexpr int kLoads = kWidth == 576 ? 9 : 8;
  const int warp = (threadIdx.x >> 5) - kConvertWarp0, lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  // Load k < 8: row `row` + 8 k, sixteen of the first 512 features; two warps share a pair of rows. Eight neighbouring lanes have rows of either parity, so that their
  // stores go to different banks (the swizzle exchanges a row's units of 16 bytes by its number). Load 8: the other 64 features of eight rows.
  const int row = 2 * (warp & 3) + (lane >> 2 & 1), box = 4 * (warp >> 2) + (lane >> 3), unit = 2 * (lane & 3);
  const int rest_row = 8 * warp + (lane >> 2);
  const int source = row * kWidth + box * 64 + unit * 8, rest_source = rest_row * kWidth + LATENT_VALUES + unit * 8;
  const uint32_t target = box * kBoxBytes + row * 128 + ((unit ^ row) << 4);
  const uint32_t rest_target = (LATENT_VALUES / 64) * kBoxBytes + rest_row * 128 + ((unit ^ (rest_row & 7)) << 4);
  uint4 raw[kLoads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) raw[k] = make_uint4(0, 0, 0, 0);
  uint32_t count = 0;
  bool given_up = false;
  Walk walk(sm);
  for (; !given_up && walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    if (piece.first == piece.last) continue;  // sees nothing
    const int32_t* table = p.table + size_t(piece.request) * p.pages;
    auto page_of = [&](int chunk) {  // lane l: the page of chunk `chunk + l`, or -1
      const int column = over(min(chunk + lane, piece.last - 1), p.by_page);
      return column < p.pages ? table[column] : -1;
    };
    int pages = page_of(piece.first);  // of 32 chunks
    // Where the chunk lies; its rows' scales, of rows `lane` and `lane` + 32; how many rows may be read.
    struct Place {
      const char* at;
      int scale_low, scale_high, valid;
    };
    auto place_of = [&](int chunk) {
      const int page = __shfl_sync(0xffffffffu, pages, (chunk - piece.first) & 31);
      Place place = {p.held, 0, 0, 0};
      if (unsigned(page) < unsigned(p.blocks)) {
        const int64_t first = int64_t(page) * p.page_rows + (chunk * kChunk - over(chunk, p.by_page) * p.page_rows);
        place.at = p.held + first * kWidth;
        place.valid = min(kChunk, piece.length - chunk * kChunk);
        place.scale_low = p.scales[(first + lane) >> p.block_shift];
        place.scale_high = p.scales[(first + lane + 32) >> p.block_shift];
      } else if (warp == 0 && lane == 0) {
        report(p.status, SPARSE_MLA_STATUS_BAD_PAGE, int(piece.row / p.heads), chunk * kChunk);
      }
      return place;
    };
    auto load = [&](const Place& place, int k) { raw[k] = load_held(place.at + (k < 8 ? source + k * 8 * kWidth : rest_source)); };
    Place next = place_of(piece.first);
    if (next.valid > 0) {
#pragma unroll
      for (int k = 0; k < kLoads; ++k) load(next, k);
    }
    for (int chunk = piece.first; chunk < piece.last; ++chunk, ++count) {
      const Place own = next;
      next.valid = 0;
      if (chunk + 1 < piece.last) {
        if (((chunk + 1 - piece.first) & 31) == 0) pages = page_of(chunk + 1);
        next = place_of(chunk + 1);
      }
      // (what is behind the request's length, or in no page, becomes zeros: as bits any byte is a finite number)
      const uint32_t low = lane < own.valid ? multiplier_of<kFormat>(own.scale_low) : 0u, high = lane + 32 < own.valid ? multiplier_of<kFormat>(own.scale_high) : 0u;
      const bool twice = __any_sync(0xffffffffu, max(own.scale_low == 255 ? 0 : own.scale_low, own.scale_high == 255 ? 0 : own.scale_high) > kMostInOne);
      const uint32_t stage = count % kStages, use = count / kStages;
      if (use > 0 && !warp_wait(sm.bar(kFree0 + stage), (use - 1) & 1, abort_flag)) { given_up = true; break; }
      unsigned char* tile = sm.ptr + stage * L::kTileBytes;
      if (warp == 0 && lane == 0) *sm.live(stage) = own.valid;
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int from = k < 8 ? (row + 8 * k) & 31 : rest_row & 31;
        const bool upper = k < 8 ? k >= 4 : warp >= 4;
        const uint32_t factor = __shfl_sync(0xffffffffu, upper ? high : low, from);
        const uint4 v = raw[k];
        uint32_t words[8] = {widened<kFormat, 0>(v.x, factor), widened<kFormat, 1>(v.x, factor), widened<kFormat, 0>(v.y, factor), widened<kFormat, 1>(v.y, factor),
                             widened<kFormat, 0>(v.z, factor), widened<kFormat, 1>(v.z, factor), widened<kFormat, 0>(v.w, factor), widened<kFormat, 1>(v.w, factor)};
        if (twice) {
          const int byte = __shfl_sync(0xffffffffu, upper ? own.scale_high : own.scale_low, from);
          const uint32_t more = second_multiplier_of<kFormat>(byte);
#pragma unroll
          for (int e = 0; e < 8; ++e) words[e] = multiply_pair<kFormat>(words[e], more);
        }
        const uint32_t at = k < 8 ? target + k * 1024 : rest_target;
        *reinterpret_cast<uint4*>(tile + at) = make_uint4(words[0], words[1], words[2], words[3]);
        *reinterpret_cast<uint4*>(tile + (at ^ 16)) = make_uint4(words[4], words[5], words[6], words[7]);
        if (next.valid > 0) load(next, k);
      }
      fence_proxy_async();  // products read the tile through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kFull0 + stage));
    }
  }
}

// A softmax thread holds a row's 32 scores twice: 144 + 72 + 72 + 96 + 96 of the warpgroups' 5 x 96 registers.
__device__ __forceinline__ void share_registers(int warp) {
  if (warp < kSoftmaxWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;\n");
  else if (warp < kConvertWarp0) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
}

// As `query_role`, with a subpartition's rows all one warp's: in three parts, so that few registers do.
template <int kWidth>
__device__ void query_role8(const Params& p, const Shared& sm, uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  const int subpartition = warp & 3;
  const uint32_t lanes = uint32_t(subpartition * 32) << 16;
  constexpr int kSegments = kWidth / 32, kParts = 3, kOwn = (kSegments + kParts - 1) / kParts;
  uint32_t loads = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    if (piece.first == piece.last) continue;  // sees nothing
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      uint4 words[2 * kOwn];
#pragma unroll
      for (int s = 0; s < kOwn; ++s) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int segment = part * kOwn + s, row = subpartition * 16 + (lane >> 2) + 8 * k;
          words[2 * s + k] = make_uint4(0, 0, 0, 0);
          if (segment < kSegments && row < piece.rows)
            words[2 * s + k] = *reinterpret_cast<const uint4*>(p.q + (piece.row + row) * (kWidth * 2) + segment * 64 + (lane & 3) * 16);
        }
      }
      if (part == 0) {
        if (loads > 0 && !warp_wait(sm.bar(kQFree), (loads - 1) & 1, abort_flag, kLongWait)) return;
        tc_fence_after_sync();
      }
#pragma unroll
      for (int s = 0; s < kOwn; ++s) {
        const int segment = part * kOwn + s;
        if (segment >= kSegments) continue;
        const uint32_t at = tmem + lanes + (segment < 16 ? kColumnsQ + segment * 8 : kColumnsQRest + (segment - 16) * 8);
        const uint4 a = words[2 * s], b = words[2 * s + 1];
        tmem_st_8(at, a.x, a.z, b.x, b.z);
        tmem_st_8(at + kHighLanes, a.y, a.w, b.y, b.w);
      }
    }
    tmem_wait_st();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.bar(kQFull));
    ++loads;
  }
}

}  // namespace absorbed
}  // namespace latent
