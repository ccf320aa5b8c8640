// Rows held in 8 bits on their way into the absorbed attention kernel's tiles (included by latent_attention.cu).
//
// A value is an e4m3 number times its block's scale, a power of two: in 16 bits the product is exact, so products, softmax and sums are those
// of a 16-bit cache that holds the same numbers. Of s.eeee.mmm the bits moved to s.0000eeee.mmm0000 are, as bfloat16, the value times
// 2^-120 (subnormal numbers too), and to s.0eeee.mmm0000000, as half, times 2^-8; one multiplication of a pair by the scale times 2^120 or 2^8 does the
// rest: a permutation, a shift, a mask and a product for two values.
//
// What bounds it: shared memory. Of the 2.7 k cycles of a chunk its ports are busy for 2.5 k: bytes in, bytes out, values over them, the two products' operands. Half queries, and
// bfloat16 ones in small calls (latent_turned8.cuh has the others). 64 requests of 64 heads at 32K 411 us, 32 x 6 at 16K 535, one token at 8K 17.5 (its 16 us are the chain
// that latent_attention.cu describes). With bytes by plain loads into registers 427 and 566, with two groups of warps in turn 459 and 589, tiles widened as a whole 431 and 568 (now
// halves: 64 keys wait for 32), quarters as halves; conversions of e4m3 to half by the converter are no faster than the four instructions.
//
//   warps 8-11   Q of the next piece from global to tensor memory (a subpartition each)
//   warp 6       brings chunks (64 rows of W bytes, contiguous) by bulk copies, and asks for the rows behind them in L2
//   warps 12-19  a group of eight of the chunk's rows each: e4m3 numbers out of shared memory, values over them
#pragma once

namespace latent {
namespace absorbed {

constexpr int kQueryWarps8 = 4, kConvertWarp0 = kQueryWarp0 + kQueryWarps8, kConvertWarps = 8;
constexpr int kThreads8 = 32 * (kConvertWarp0 + kConvertWarps);

// A scale's byte: 2^(byte - 127), 255: NaN. The multiplier (twice, for a pair) is 2^(byte - kBias); what is above the type's largest power of two is
// left for a second one. With NaN the values are zeros and the scores become NaN, for as values NaN would reach all rows of a tile, by weights of zero too.
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
  if (byte == 255) return 0u;
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

__device__ __forceinline__ void store_shared(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
// Global to shared memory (16-byte aligned, a multiple of 16 bytes); counts its bytes on `bar`.
__device__ __forceinline__ void bulk_copy(uint32_t target, const char* source, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(target), "l"(source), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_prefetch(const char* source, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(source), "r"(bytes) : "memory");
}

// Eight rows of a tile (a group) lie together: their boxes of 64 features one after the other, each 1024 bytes as the products want them. Before that the rows' 8-bit
// numbers lie in the upper half of the same memory.
template <int kWidth> constexpr int kGroupBytes = kWidth / 64 * 1024;
template <int kWidth> constexpr int kHeldBytes = kWidth * 8;
static_assert(kGroupBytes<576> == 2 * kHeldBytes<576> && kGroupBytes<512> == 2 * kHeldBytes<512>, "the numbers fill half of what their values do");
constexpr int kAhead = 4;  // chunks whose rows are on their way to L2

template <int kWidth>
__device__ void copy_role8(const Params& p, const Shared& sm) {
  using L = Layout<kWidth>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0;
  bool given_up = false, half_given = false;
  Walk walk(sm);
  for (; !given_up && walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    if (piece.first == piece.last) continue;  // sees nothing
    const int32_t* table = p.table + size_t(piece.request) * p.pages;
    // Lane l: the first row of chunk `chunk + l` in the cache, or -1.
    auto rows_of = [&](int chunk) {
      const int own = min(chunk + lane, piece.last - 1), column = over(own, p.by_page);
      const int page = column < p.pages ? table[column] : -1;
      return unsigned(page) < unsigned(p.blocks) ? int64_t(page) * p.page_rows + (own * kChunk - column * p.page_rows) : int64_t(-1);
    };
    auto valid_of = [&](int chunk) { return min(kChunk, piece.length - chunk * kChunk); };
    int64_t rows = 0, next_rows = rows_of(piece.first);  // of 32 chunks; of the next 32
    for (int chunk = piece.first; chunk < piece.last; ++chunk, ++count) {
      const int place = (chunk - piece.first) & 31;
      if (place == 0) {
        rows = next_rows;
        if (chunk + 32 < piece.last) next_rows = rows_of(chunk + 32);
        if (lane < kAhead && chunk + lane < piece.last && rows >= 0) bulk_prefetch(p.held + rows * kWidth, valid_of(chunk + lane) * kWidth);
      }
      // (the first chunks of a window are asked for above)
      if (place + kAhead < 32 && lane == place + kAhead && chunk + kAhead < piece.last && rows >= 0) bulk_prefetch(p.held + rows * kWidth, valid_of(chunk + kAhead) * kWidth);
      const int64_t first = __shfl_sync(0xffffffffu, rows, place);
      const int valid = first >= 0 ? valid_of(chunk) : 0;
      int low = 0, high = 0;
      if (first >= 0) {
        low = p.scales[(first + lane) >> p.block_shift];
        high = p.scales[(first + lane + 32) >> p.block_shift];
      }
      const uint32_t stage = count % kStages, use = count / kStages, target = sm.base + stage * L::kTileBytes + lane * kGroupBytes<kWidth> + kHeldBytes<kWidth>;
      const char* source = p.held + (first + lane * 8) * kWidth;
      const int own = min(max(valid - lane * 8, 0), 8);  // rows of group `lane`
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // (the first four groups' memory is free earlier)
        const uint32_t bar = sm.bar(kLanded0 + 2 * stage + half);
        if (use > 0 && !warp_wait(sm.bar((half ? kFree0 : kFreeHalf0) + stage), (use - 1) & 1, abort_flag)) {
          given_up = true;
          half_given = half == 1;
          break;
        }
        if (half == 0) {
          // (what the chunk before says has been read: its second product has begun)
          if (lane == 0) {
            *sm.live(stage) = valid;
            if (first < 0) report(p.status, SPARSE_MLA_STATUS_BAD_PAGE, int(piece.row / p.heads), chunk * kChunk);
          }
          unsigned char* scales = sm.ptr + L::kSmemScales + stage * kChunk;
          scales[lane] = static_cast<unsigned char>(low);
          scales[lane + 32] = static_cast<unsigned char>(high);
          __syncwarp();
        }
        if (half == 1) {  // (nobody waits for this yet)
          const uint32_t spoilt[2] = {__ballot_sync(0xffffffffu, low == 255 && lane < valid), __ballot_sync(0xffffffffu, high == 255 && lane + 32 < valid)};
          if (lane == 0) {
            *sm.marked(stage) = (spoilt[0] | spoilt[1]) != 0 ? valid - kSpoilt : valid;
            *sm.spoilt(stage, 0) = spoilt[0];
            *sm.spoilt(stage, 1) = spoilt[1];
          }
        }
        if (lane == 0) mbar_arrive_expect(bar, min(max(valid - half * 32, 0), 32) * kWidth);
        __syncwarp();
        if (lane >> 2 == half && own > 0) bulk_copy(target, source, own * kWidth, bar);
      }
      if (given_up) break;
    }
  }
  if (*abort_flag != 0) {  // nothing of this block may be written behind its end
    int never = 0;
    for (uint32_t i = count > kStages ? count - kStages : 0; i < count; ++i)
      for (int half = 0; half < 2; ++half) mbar_wait(sm.bar(kLanded0 + 2 * (i % kStages) + half), (i / kStages) & 1, &never);
    if (half_given) mbar_wait(sm.bar(kLanded0 + 2 * (count % kStages)), (count / kStages) & 1, &never);
  }
}

// A warp to each group: its numbers to registers, and as values over the memory that they lay in.
template <int kFormat, int kWidth>
__device__ void convert_role(const Params& p, const Shared& sm) {
  using L = Layout<kWidth>;
  constexpr int kLoads = kWidth == 576 ? 9 : 8;
  const int group = (threadIdx.x >> 5) - kConvertWarp0, lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  // Load k < 8: of row 2 (k / 2) + `odd` sixteen features of its half number k % 2. Eight neighbouring lanes have rows of either parity, so that their stores go to
  // different banks (the swizzle exchanges a row's units of 16 bytes by its number), and 64 bytes in different halves of 128 for the loads. Load 8: the other
  // 64 features of all rows.
  const int odd = lane >> 2 & 1, unit = 2 * (lane & 3), box = lane >> 3 ^ (kWidth == 512 ? odd : 0), rest_row = lane >> 2;
  const uint32_t base = sm.base + group * kGroupBytes<kWidth>;
  const uint32_t source = base + kHeldBytes<kWidth> + odd * kWidth + box * 64 + unit * 8, rest_source = base + kHeldBytes<kWidth> + rest_row * kWidth + LATENT_VALUES + unit * 8;
  const uint32_t target = base + box * 1024 + odd * 128 + ((unit ^ odd) << 4), rest_target = base + LATENT_VALUES / 64 * 1024 + rest_row * 128 + ((unit ^ rest_row) << 4);
  uint32_t count = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    for (int left = walk.piece.last - walk.piece.first; left > 0; --left, ++count) {
      const uint32_t stage = count % kStages, tile = stage * L::kTileBytes;
      if (!warp_wait(sm.bar(kLanded0 + 2 * stage + (group >> 2)), (count / kStages) & 1, abort_flag)) return;
      const int byte = sm.ptr[L::kSmemScales + stage * kChunk + group * 8 + (lane & 7)], live = *sm.live(stage);
      uint4 raw[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k) raw[k] = load_shared(tile + (k < 8 ? source + (k >> 1) * 2 * kWidth + (k & 1) * 256 : rest_source));
      // What is behind the request's length, or in no page, becomes zeros: as bits any byte is a finite number.
      const uint32_t own = group * 8 + (lane & 7) < live ? multiplier_of<kFormat>(byte) : 0u;
      const bool twice = __any_sync(0xffffffffu, byte != 255 && byte > kMostInOne);  // (scales above 2^7)
      const uint32_t more = twice ? second_multiplier_of<kFormat>(byte) : 0u;
      auto widen = [&](int k) {
        const int row = k < 8 ? 2 * (k >> 1) + odd : rest_row;
        const uint32_t factor = __shfl_sync(0xffffffffu, own, row);
        const uint32_t to = tile + (k < 8 ? (target ^ (k >> 1) << 5) + (k >> 1) * 256 + (k & 1) * 4096 : rest_target);
        uint32_t words[8] = {widened<kFormat, 0>(raw[k].x, factor), widened<kFormat, 1>(raw[k].x, factor), widened<kFormat, 0>(raw[k].y, factor), widened<kFormat, 1>(raw[k].y, factor),
                             widened<kFormat, 0>(raw[k].z, factor), widened<kFormat, 1>(raw[k].z, factor), widened<kFormat, 0>(raw[k].w, factor), widened<kFormat, 1>(raw[k].w, factor)};
        if (twice) {
          const uint32_t again = __shfl_sync(0xffffffffu, more, row);
#pragma unroll
          for (int e = 0; e < 8; ++e) words[e] = multiply_pair<kFormat>(words[e], again);
        }
        store_shared(to, words[0], words[1], words[2], words[3]);
        store_shared(to ^ 16, words[4], words[5], words[6], words[7]);
      };
#pragma unroll
      for (int k = 0; k < 8; k += 2) widen(k);  // to the lower half of the group's memory
      __syncwarp();  // all of its numbers are in registers
#pragma unroll
      for (int k = 1; k < 8; k += 2) widen(k);
      if constexpr (kLoads > 8) widen(8);
      fence_proxy_async();  // products read the tile through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kFull0 + stage));
    }
  }
}

// Of the warpgroups' 5 x 96 registers a softmax thread has 128, one that brings chunks 112, the others 64. (Each at the head of its role's branch.)
__device__ __forceinline__ void take_128_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 128;\n"); }
__device__ __forceinline__ void take_112_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 112;\n"); }
__device__ __forceinline__ void keep_64_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n"); }

// As `query_role`, with a subpartition's rows all one warp's: in four parts, so that few registers do.
template <int kWidth>
__device__ void query_role8(const Params& p, const Shared& sm, uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  const int subpartition = warp & 3;
  const uint32_t lanes = uint32_t(subpartition * 32) << 16;
  constexpr int kSegments = kWidth / 32, kParts = 4, kOwn = (kSegments + kParts - 1) / kParts;
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
