// Attention of prompts in expanded form: keys and values per head, and one rope key per token for all heads.
//
// out = softmax(scale q . [k | k_rope]) v per head, causal or not, over ragged requests. One block takes 256 query rows of a
// head as two tiles of 128 and walks the keys in tiles of 128. All products run on tcgen05 with M = 128, N = 128: S = Q K^T from shared
// memory (K = 192), O += P V with P from tensor memory (K = 128). While the softmax warps of one tile work, the products of
// the other run.
//
//   warps 0-3, 4-7  softmax of tile 0 and 1: a thread owns a query row. Scores out of tensor memory, running reference and
//                   sum in FP32, P (16 bits) over the scores' columns, output.
//   warp 8          one thread issues the products.
//   warp 9          one thread brings boxes of 64 features x 128 rows (16 KiB) by tensor copies into a ring of eight:
//                   three of a key tile (128 features of the head, 64 of rope), two of a value tile, in the order of their use.
//   warp 10         finds out what the block does next: blocks that have not started yet are taken over, one after the other, by those
//                   that run (cluster launch control). The copies and first products of the next 256 rows run beside the output of the last.
//
// Tensor memory: scores (P over their first half) of tile t in columns 128 t .. + 127, O of tile t in 256 + 128 t .. + 127.
//
// What paces it: a tile's chain of scores to weights (about 1.9 k cycles: 128 exponentials per thread at 8 cycles a warp are 1.0 k of them) and products
// (1.6 k, of which 1.3 k are the tensor core's), 3.8 k per step of both tiles against 2.6 k of products. In a loop of large calls the
// board's power limit, not the chain, decides: 8192 x 8192 tokens of 64 heads, causal, take 1.13 ms in a few calls after a pause (1.22 PFLOP/s) and
// 1.20 to 1.25 ms in a long loop (1.10 to 1.14 PFLOP/s, 1.6 GHz), and what shortens the chain gives a third of that there. Before: one block per 256 rows and
// a maximum for every step 1.29 ms; a quarter of the exponentials by a polynomial, weights handed over in halves, and the rows of two heads
// in a block where a request has no more than 128 were no faster or slowed the large calls down. Registers decide: 160 bytes of spills in the softmax
// loop make 1.39 ms of it.
//
// Rows of a value box behind the request's last key are cleared before they are multiplied: their weights are zero, but they
// belong to other requests (or to nobody) and 0 x infinity would be a NaN. Scores of such keys are replaced, whatever they are.
#include "latent_common.cuh"
#include "latent_parts.cuh"
#include "latent_ptx.cuh"

namespace latent {
namespace prefill {

using namespace sm100;

constexpr int kTile = 128;                    // query rows of a tile, keys of a step
constexpr int kFeatures = LATENT_NOPE + LATENT_ROPE;
constexpr int kThreads = 384;  // (the last warp has nothing to do but to give registers away)
constexpr int kSoftmaxWarps = 8, kProductWarp = 8, kCopyWarp = 9, kPlanWarp = 10;
constexpr int kBoxBytes = kTile * 128;        // 64 features of 128 rows
constexpr int kQBoxes = kFeatures / 64, kKeyBoxes = 3, kValueBoxes = 2, kRing = 8;
constexpr int kItems = 2;                     // announced ahead

// A call of few items leaves SMs without work, so items of many steps are cut into pieces there (for all SMs, no piece shorter than kLeastSteps), and
// `join_kernel` adds up what they leave. The sums' way through memory and the second launch take 13 us, a step 2: not where the longest item is
// not shortened by kSavedSteps. (16 heads, whole / cut: 512 queries at 2048 keys 39 / 27 us, at 16384 255 / 85-95, 1024 at 8192 134 / 88-94, one at
// 131072 1890 / 241-264; five steps saved, 256 at 1025, 26 / 30. A call of few items whose requests turn out too short pays 3 us for the launch.)
constexpr int kItemRows = 2 * kTile, kLeastSteps = 4, kSavedSteps = 8;
constexpr int kSlotFloats = kItemRows * LATENT_NOPE;

constexpr int kSmemQ = 0;                                       // two tiles of three boxes
constexpr int kSmemRing = kSmemQ + 2 * kQBoxes * kBoxBytes;
constexpr int kSmemBars = kSmemRing + kRing * kBoxBytes;
constexpr int kSmemMisc = kSmemBars + 320;                       // tensor-memory slot, abort flag; 32: answer of the launch control; 64: items
constexpr int kSmemEnd = kSmemMisc + 64 + kItems * 32;
constexpr int kSmemBytes = kSmemEnd + 1024;                     // the tiles are aligned to 1024 bytes

constexpr uint32_t kColumnsO = 256;

enum Bar {
  kFull0 = 0, kFree0 = kRing, kQFull0 = 2 * kRing, kQFree0 = kQFull0 + 2, kScores0 = kQFree0 + 2, kWeights0 = kScores0 + 2, kOut0 = kWeights0 + 2,
  kMended = kOut0 + 2, kAnswer, kNearlyDone, kItemReady0, kGivenUp = kItemReady0 + kItems, kItemDone0, kBarCount = kItemDone0 + kItems
};
static_assert(kBarCount <= 40, "the barrier area");

struct Params {
  CUtensorMap q, k, v, rope;
  const int32_t *cu_q, *cu_k;
  void* out;
  float* lse;
  int32_t* status;
  int32_t batches, tokens, keys, heads, q_head, k_head, v_head;  // *_head: 0 where all heads share memory
  int32_t causal;
  int32_t sectors;    // rows of `out` begin on 32-byte boundaries (otherwise on 16-byte ones)
  int32_t slots;      // of the workspace, one for every piece; 0: items are whole
  float2* statistics; // [slots, 256]
  float* sums;        // [slots], see sums_place
  float scale_log2;
};
// Sums of eight features of 32 rows lie next to each other, as warps write them. First feature of eight.
__device__ __forceinline__ int sums_place(int row, int feature) { return (((row >> 5) * (LATENT_NOPE / 8) + feature / 8) * 32 + (row & 31)) * 8; }

struct Shared {
  uint32_t base;
  unsigned char* ptr;
  __device__ __forceinline__ uint32_t bar(int which) const { return base + kSmemBars + which * 8; }
  __device__ __forceinline__ uint32_t* slot() const { return reinterpret_cast<uint32_t*>(ptr + kSmemMisc); }
  __device__ __forceinline__ volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(ptr + kSmemMisc + 4); }
  __device__ __forceinline__ uint32_t answer() const { return base + kSmemMisc + 32; }
  __device__ __forceinline__ struct Item* item(uint32_t index) const;
};

// 256 query rows of a head.
struct Item {
  int head;
  int row;    // first query token
  int rows;   // query rows
  int first;  // first key of the request
  int keys;   // keys that the request has
  int offset; // row i sees keys below offset + i + 1 (causal)
  int slot;   // -1: the item is whole; >= 0: a piece, whose sums go there; kNoPiece: there is nothing to do
};
constexpr int kNoPiece = -2;
static_assert(sizeof(Item) <= 32, "the item ring holds 32-byte entries");
__device__ __forceinline__ Item* Shared::item(uint32_t index) const { return reinterpret_cast<Item*>(ptr + kSmemMisc + 64 + index % kItems * 32); }

// Keys that the first `rows` rows of the item see, at most.
__device__ __forceinline__ int reach(const Params& p, const Item& item, int rows) {
  if (rows <= 0) return 0;
  return p.causal ? min(item.keys, max(0, item.offset + rows)) : item.keys;
}

// Key steps of tile t.
__device__ __forceinline__ int steps_of(const Params& p, const Item& item, int t) {
  return item.rows <= t * kTile ? 0 : (reach(p, item, min(item.rows, (t + 1) * kTile)) + kTile - 1) / kTile;
}

// How a call's items are cut: up to `pieces` of each, of `steps` key steps; pieces == 1: not at all.
struct Cut {
  int pieces, steps;
  __device__ __forceinline__ int of(const Params& p, const Item& item) const { return max((max(steps_of(p, item, 0), steps_of(p, item, 1)) + steps - 1) / steps, 1); }
};

// Item number `index` (whole), by whole warps; false when there are fewer. Items: heads, of each all requests, of each request blocks of
// 256 rows from its end (where causal rows see most keys) to its beginning. With kPieces, `index` counts pieces,
// as many for each item as the call's longest may be cut into.
template <bool kPieces>
__device__ __forceinline__ bool find_whole(const Params& p, int index, Item& item, Cut* cut) {
  const int lane = threadIdx.x & 31;
  int per_head = 0, most_keys = 0;
  for (int b = lane; b < p.batches; b += 32) {
    const int blocks = (max(bounded(fetch(p.cu_q + b + 1), p.tokens) - bounded(fetch(p.cu_q + b), p.tokens), 0) + 255) >> 8;
    per_head += blocks;
    if (kPieces && blocks > 0) most_keys = max(most_keys, bounded(fetch(p.cu_k + b + 1), p.keys) - bounded(fetch(p.cu_k + b), p.keys));
  }
  per_head = __reduce_add_sync(0xffffffffu, per_head);
  if (per_head == 0) return false;
  if (kPieces) {
    const int most = (__reduce_max_sync(0xffffffffu, most_keys) + kTile - 1) / kTile, pieces = max(p.slots / p.heads / per_head, 1);
    cut->steps = max((most + pieces - 1) / pieces, kLeastSteps);
    cut->pieces = most - cut->steps >= kSavedSteps ? pieces : 1;
    index /= cut->pieces;
  }
  if (index / per_head >= p.heads) return false;
  item.head = index / per_head;
  int left = index - item.head * per_head;
  for (int first = 0;; first += 32) {  // (ends: left < per_head)
    const int b = first + lane;
    const int begin = b < p.batches ? bounded(fetch(p.cu_q + b), p.tokens) : 0;
    const int count = b < p.batches ? max(bounded(fetch(p.cu_q + b + 1), p.tokens) - begin, 0) : 0;
    const int blocks = (count + 255) >> 8;
    int before = blocks;  // inclusive prefix sum
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += other;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, left < before);
    if (hit == 0) {
      left -= __shfl_sync(0xffffffffu, before, 31);
      continue;
    }
    const int owner = __ffs(hit) - 1;
    const int k_begin = b < p.batches ? bounded(fetch(p.cu_k + b), p.keys) : 0;
    const int k_count = b < p.batches ? max(bounded(fetch(p.cu_k + b + 1), p.keys) - k_begin, 0) : 0;
    const int block = __shfl_sync(0xffffffffu, before - 1 - left, owner);  // from the request's end
    const int request_count = __shfl_sync(0xffffffffu, count, owner), start = block << 8;
    item.row = __shfl_sync(0xffffffffu, begin, owner) + start;
    item.rows = min(256, request_count - start);
    item.first = __shfl_sync(0xffffffffu, k_begin, owner);
    item.keys = __shfl_sync(0xffffffffu, k_count, owner);
    item.offset = item.keys - request_count + start;
    item.slot = -1;
    return true;
  }
}

// What block `index` does: an item, or a piece of one, which is the item as it would be if its keys began and ended with the piece's.
template <bool kPieces>
__device__ __forceinline__ bool find_item(const Params& p, int index, Item& item) {
  Cut cut;
  if (!find_whole<kPieces>(p, index, item, &cut)) return false;
  if (kPieces && cut.pieces > 1) {
    const int count = cut.of(p, item), piece = index % cut.pieces, keys = cut.steps * kTile;  // (of a piece)
    if (piece >= count) {
      item.slot = kNoPiece;
      item.keys = 0;
    } else if (count > 1) {
      item.slot = index;
      item.first += piece * keys;
      item.offset -= piece * keys;
      item.keys = min(item.keys - piece * keys, keys);
    }
  }
  return true;
}

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit = 1ll << 31) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit));
}

// ---- what to do next ------------------------------------------------------------------------------------------------

// Asks for a block of the launch that has not started; 16 bytes at `answer` and on `bar` in time. Not after a refusal.
__device__ __forceinline__ void ask_for_block(uint32_t answer, uint32_t bar) {
  mbar_arrive_expect(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(answer), "r"(bar) : "memory");
}
// The block that was given (it will not start), or -1.
__device__ __forceinline__ int block_given(uint32_t answer) {
  uint32_t given, index;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b128 r;\n"
      "ld.shared.b128 r, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "mov.u32 %1, 0;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, r;\n"
      "}\n"
      : "=r"(given), "=r"(index) : "r"(answer) : "memory");
  return given != 0 ? int(index) : -1;
}

// By a whole warp. `item` is the first.
template <bool kPieces>
__device__ void plan_role(const Params& p, const Shared& sm, Item item) {
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  uint32_t announced = 0, asked = 0;
  for (bool has = true;; ) {
    if (announced >= kItems && !warp_wait(sm.bar(kItemDone0 + announced % kItems), (announced / kItems - 1) & 1, abort_flag, kLongWait)) return;
    if (lane == 0) {
      Item* target = sm.item(announced);
      *target = item;
      if (!has) target->rows = 0;  // no more
      mbar_arrive(sm.bar(kItemReady0 + announced % kItems));
    }
    ++announced;
    if (!has) return;
    // The next block is asked for when the copies of this item's last step but one begin: early enough for the answer to come in time, no earlier, so
    // that the last items go to whoever is free (8192 x 8192 tokens, 64 heads: asked for with the item's announcement 1389 us, so 1289).
    if (!warp_wait(sm.bar(kNearlyDone), asked & 1, abort_flag, kLongWait)) return;
    if (lane == 0) {
      fence_proxy_async();  // (the answer before was read through the generic proxy)
      ask_for_block(sm.answer(), sm.bar(kAnswer));
    }
    // (also where a wait has given up: the answer is still to come)
    int never = 0;
    if (!__all_sync(0xffffffffu, mbar_wait(sm.bar(kAnswer), asked & 1, &never))) *abort_flag = 1;
    ++asked;
    if (*abort_flag != 0) return;
    int index = block_given(sm.answer());
    __syncwarp();
    has = index >= 0 && find_item<kPieces>(p, index, item);
    if (!has) {
      // Numbers grow: the blocks behind this one have nothing to do either. They are taken over so that they need not start.
      while (index >= 0) {
        if (lane == 0) {
          fence_proxy_async();
          ask_for_block(sm.answer(), sm.bar(kAnswer));
        }
        if (!__all_sync(0xffffffffu, mbar_wait(sm.bar(kAnswer), asked & 1, &never))) { *abort_flag = 1; return; }
        ++asked;
        index = block_given(sm.answer());
        __syncwarp();
      }
    }
  }
}

// Everybody's way through the items.
struct Walk {
  const Shared& sm;
  uint32_t index = 0;
  Item item;
  __device__ __forceinline__ explicit Walk(const Shared& shared) : sm(shared) {}
  __device__ __forceinline__ bool read() { item = *sm.item(index); return item.rows > 0; }
  __device__ __forceinline__ int slot() const { return *static_cast<volatile int*>(&sm.item(index)->slot); }  // (read where it is wanted: registers are scarce)
  __device__ __forceinline__ bool next_of_warp() { return warp_wait(sm.bar(kItemReady0 + index % kItems), (index / kItems) & 1, sm.abort_flag(), kLongWait) && read(); }
  __device__ __forceinline__ bool next_of_thread() { return mbar_wait(sm.bar(kItemReady0 + index % kItems), (index / kItems) & 1, sm.abort_flag(), kLongWait) && read(); }
  __device__ __forceinline__ void done() { mbar_arrive(sm.bar(kItemDone0 + index % kItems)); ++index; }
  __device__ __forceinline__ void done_of_warp() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(sm.bar(kItemDone0 + index % kItems));
    ++index;
  }
};

// ---- copies ---------------------------------------------------------------------------------------------------------

// By the whole warp; lane 0 issues.
__device__ void copy_role(const Params& p, const Shared& sm) {
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0, mended = 0, loads[2] = {0, 0};  // boxes so far; those that were cleared in part; tiles of Q
  bool given_up = false;
  // Claims the next slot of the ring and lets its copy be started by lane 0.
  auto bring = [&](auto start, int valid_rows) {
    const uint32_t slot = count % kRing, use = count / kRing, target = sm.base + kSmemRing + slot * kBoxBytes;
    if (use > 0 && !warp_wait(sm.bar(kFree0 + slot), (use - 1) & 1, abort_flag)) { given_up = true; return; }
    const bool mend = valid_rows < kTile;
    const uint32_t bar = sm.bar(mend ? int(kMended) : int(kFull0 + slot));
    if (lane == 0) {
      mbar_arrive_expect(bar, kBoxBytes);
      start(target, bar);
    }
    __syncwarp();
    if (mend) {
      if (!warp_wait(bar, mended++ & 1, abort_flag)) { given_up = true; return; }
      // (the swizzle stays within a row)
      for (int at = valid_rows * 128 + lane * 16; at < kBoxBytes; at += 512)
        *reinterpret_cast<uint4*>(sm.ptr + kSmemRing + slot * kBoxBytes + at) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kFull0 + slot));
    }
    ++count;
  };
  Walk walk(sm);
  for (; !given_up && walk.next_of_warp(); walk.done_of_warp()) {
    const Item& item = walk.item;
    const int steps_0 = steps_of(p, item, 0), steps_1 = steps_of(p, item, 1), steps = max(steps_0, steps_1);
    if (steps == 0 && lane == 0) mbar_arrive(sm.bar(kNearlyDone));
    for (int step = 0; step < steps && !given_up; ++step) {
      if (step == max(steps - 2, 0) && lane == 0) mbar_arrive(sm.bar(kNearlyDone));
      const int key = item.first + step * kTile;
      for (int box = 0; box < 2 && !given_up; ++box)
        bring([&](uint32_t target, uint32_t bar) { copy_box(target, &p.k, box * 64, item.head * p.k_head, key, bar); }, kTile);
      if (!given_up) bring([&](uint32_t target, uint32_t bar) { copy_box(target, &p.rope, 0, key, bar); }, kTile);
#pragma unroll
      for (int t = 0; t < 2; ++t) {  // (rows behind the item are multiplied and thrown away)
        if (step > 0 || given_up || (t == 0 ? steps_0 : steps_1) == 0) continue;
        if (loads[t] > 0 && !warp_wait(sm.bar(kQFree0 + t), (loads[t] - 1) & 1, abort_flag)) { given_up = true; continue; }
        if (lane == 0) {
          mbar_arrive_expect(sm.bar(kQFull0 + t), kQBoxes * kBoxBytes);
#pragma unroll
          for (int box = 0; box < kQBoxes; ++box)
            copy_box(sm.base + kSmemQ + (t * kQBoxes + box) * kBoxBytes, &p.q, box * 64, item.head * p.q_head, item.row + t * kTile, sm.bar(kQFull0 + t));
        }
        __syncwarp();
        ++loads[t];
      }
      const int valid = min(kTile, item.keys - step * kTile);
      for (int box = 0; box < kValueBoxes && !given_up; ++box)
        bring([&](uint32_t target, uint32_t bar) { copy_box(target, &p.v, box * 64, item.head * p.v_head, key, bar); }, valid);
    }
  }
  if (*abort_flag != 0) {  // nothing of this block may be written behind its end
    int never = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (loads[t] > 0) mbar_wait(sm.bar(kQFull0 + t), (loads[t] - 1) & 1, &never);
    for (uint32_t i = count > kRing ? count - kRing : 0; i < count; ++i) mbar_wait(sm.bar(kFull0 + i % kRing), (i / kRing) & 1, &never);
    if (mended > 0) mbar_wait(sm.bar(kMended), (mended - 1) & 1, &never);
  }
}

// ---- products (one thread) -------------------------------------------------------------------------------------------

template <int kFormat> constexpr uint32_t kIdescScores = idesc_f16(128, 128, kFormat, 0, 0);
template <int kFormat, int kColumns> constexpr uint32_t kIdescValues = idesc_f16(128, kColumns, kFormat, 0, 1);

template <int kFormat>
__device__ void product_role(const Params& p, const Shared& sm, uint32_t tmem) {
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0, loads[2] = {0, 0}, weights_seen[2] = {0, 0};  // boxes used; tiles of Q; weights
  auto box_at = [&](uint32_t box) { return sm.base + kSmemRing + box % kRing * kBoxBytes; };
  auto landed = [&](uint32_t box) { return mbar_wait(sm.bar(kFull0 + box % kRing), (box / kRing) & 1, abort_flag); };
  auto release = [&](uint32_t first, int boxes) {
    for (int i = 0; i < boxes; ++i) mma_commit(sm.bar(kFree0 + (first + i) % kRing));
  };
  auto scores = [&](int t, uint32_t keys) {
#pragma unroll
    for (int box = 0; box < kKeyBoxes; ++box) {
      const uint64_t a = smem_desc_sw128(sm.base + kSmemQ + (t * kQBoxes + box) * kBoxBytes, 16, 1024);
      const uint64_t b = smem_desc_sw128(box_at(keys + box), 16, 1024);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (box == 0 && k == 0) mma_ss_c<false>(tmem + t * kTile, a, b, kIdescScores<kFormat>);
        else mma_ss_c<true>(tmem + t * kTile, a + k * 2, b + k * 2, kIdescScores<kFormat>);
      }
    }
    mma_commit(sm.bar(kScores0 + t));
  };
  auto keys_landed = [&](uint32_t keys) { return landed(keys) && landed(keys + 1) && landed(keys + 2); };
  Walk walk(sm);
  for (; walk.next_of_thread(); walk.done()) {
    const int steps[2] = {steps_of(p, walk.item, 0), steps_of(p, walk.item, 1)};
    const int most = max(steps[0], steps[1]);
    if (most == 0) continue;
    if (!keys_landed(count)) return;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (steps[t] == 0) continue;
      if (!mbar_wait(sm.bar(kQFull0 + t), loads[t]++ & 1, abort_flag)) return;
      tc_fence_after_sync();
      scores(t, count);
      if (steps[t] == 1) mma_commit(sm.bar(kQFree0 + t));
    }
    release(count, kKeyBoxes);
    count += kKeyBoxes;
    for (int step = 0; step < most; ++step) {
      const uint32_t values = count, keys = count + kValueBoxes;
      const bool more = step + 1 < most;
      if (!landed(values) || !landed(values + 1)) return;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (step < steps[t]) {
          if (!mbar_wait(sm.bar(kWeights0 + t), weights_seen[t]++ & 1, abort_flag)) return;
          tc_fence_after_sync();
          const uint32_t o = tmem + kColumnsO + t * kTile, weights = tmem + t * kTile;
          const uint64_t b = smem_desc_sw128(box_at(values), kBoxBytes, 1024);
          if (box_at(values + 1) > box_at(values)) {
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) mma_ts(o, weights + k * 8, b + k * 128, kIdescValues<kFormat, 128>, step > 0 || k > 0);
          } else {  // every eighth time the second box is at the ring's beginning: 64 features each, which takes half as long again
            const uint64_t b1 = smem_desc_sw128(box_at(values + 1), kBoxBytes, 1024);
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) mma_ts(o, weights + k * 8, b + k * 128, kIdescValues<kFormat, 64>, step > 0 || k > 0);
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) mma_ts(o + 64, weights + k * 8, b1 + k * 128, kIdescValues<kFormat, 64>, step > 0 || k > 0);
          }
          if (step + 1 == steps[t]) mma_commit(sm.bar(kOut0 + t));
        }
        if (t == 1) release(values, kValueBoxes);
        if (step + 1 < steps[t]) {
          if (!keys_landed(keys)) return;
          scores(t, keys);
          if (step + 2 == steps[t]) mma_commit(sm.bar(kQFree0 + t));
        }
      }
      if (more) release(keys, kKeyBoxes);
      count += kValueBoxes + (more ? kKeyBoxes : 0);
    }
  }
}

// ---- softmax ----------------------------------------------------------------------------------------------------------

// A row's reference (log2) starts kFirst below the maximum of its first scores (latent_attention.cu has the reason). It moves, to kStep below the maximum of a
// step, where the step's weights sum up to more than kMostWeight: up to that sum weights fit IEEE half, and the accumulator is rarely rescaled. (A sum that
// large has a weight of more than 2^kStep in it, so that it does move.) The lower the first reference, the sooner it moves, so that with IEEE
// half all scores of the first step are looked at: 4096 x 4096 tokens of 32 heads, scores of a deviation of 1, 2, 3, 8: 190, 201, 210, 287 us, with the
// reference at the maximum of the first 32 scores 190, 201, 207, 294, with that less 8 190, 220, 237, 295.
constexpr float kStep = 8.f, kMostWeight = 61440.f;
template <int kFormat> constexpr float kFirst = kFormat == 1 ? 0.f : 6.f;
template <int kFormat> constexpr int kFirstLook = kFormat == 1 ? 1 : 4;  // parts of 32 scores
static_assert(kTile * 256 <= kMostWeight && kMostWeight < 65504.f, "the smallest sum that is looked into, and the largest weight");

template <int kFormat, bool kPieces>
__device__ void softmax_role(const Params& p, const Shared& sm, uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = warp >> 2;
  volatile int* abort_flag = sm.abort_flag();
  const int row = t * kTile + (warp & 3) * 32 + lane;  // of an item
  const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
  const uint32_t s_tmem = tmem + t * kTile + lanes, o_tmem = tmem + kColumnsO + t * kTile + lanes;
  uint32_t scores_seen = 0, outputs = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    const Item& item = walk.item;
    const int steps = steps_of(p, item, t);
    const int end = p.causal ? min(item.keys, item.offset + row + 1) : item.keys;  // this row sees keys below
    const int warp_end = p.causal ? min(item.keys, item.offset + (row & ~31) + 1) : item.keys;  // all rows of the warp see keys below
    float reference = -INFINITY, sum = 0.f;
    for (int step = 0; step < steps; ++step) {
      if (!warp_wait(sm.bar(kScores0 + t), scores_seen++ & 1, abort_flag)) return;
      tc_fence_after_sync();
      const int key = step * kTile;
      const bool masked = key + kTile > warp_end;
      uint32_t words[kTile / 2];
      float own;
      // Weights are worked out with the reference as it is, without looking for the maximum: as long as their sum stays below kMostWeight so does
      // each of them. Where it does not (for some row of the warp) the reference may move, and they are worked out again. A row's first reference comes
      // from the maximum of its first 32 or 128 scores.
      for (int look = step == 0 ? kFirstLook<kFormat> : 0;; look = 4) {  // parts of 32 scores to look at
        float2 s[2][16];  // 32 scores, and the next 32 on their way
        auto load = [&](int part) { tmem_ld32(s_tmem + part * 32, reinterpret_cast<uint32_t*>(&s[part & 1][0])); };
        auto mask = [&](int part) {
          const int seen = end - key - part * 32;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (2 * i >= seen) s[part & 1][i].x = -INFINITY;
            if (2 * i + 1 >= seen) s[part & 1][i].y = -INFINITY;
          }
        };
        if (look > 0) {
          float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int part = 0; part < 4; ++part) {
            if (part >= look) break;
            load(part);
            tmem_wait_ld();
            if (masked) mask(part);
#pragma unroll
            for (int i = 0; i < 16; ++i) most[i & 3] = greatest(most[i & 3], s[part & 1][i].x, s[part & 1][i].y);
          }
          const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale_log2;  // scale > 0
          const bool moves = top > reference + kStep;
          float alpha = 1.f;
          if (moves) {
            const float next = top - (reference == -INFINITY ? kFirst<kFormat> : kStep);
            alpha = exp2f(reference - next);
            reference = next;
          }
          sum *= alpha;
          if (step > 0 && __any_sync(0xffffffffu, moves)) {  // (scores of this step are there: the products of the one before have ended)
#pragma unroll 1
            for (int c = 0; c < kTile; c += 32) {
              uint32_t o[32];
              tmem_ld32(o_tmem + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(o_tmem + c, o);
            }
            tmem_wait_st();
          }
        }
        const float shift = reference == -INFINITY ? 0.f : -reference;
        const float2 scale = make_float2(p.scale_log2, p.scale_log2), shifts = make_float2(shift, shift);
        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        load(0);
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          tmem_wait_ld();
          if (part < 3) load(part + 1);
          if (masked) mask(part);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 weight = fma2(s[part & 1][i], scale, shifts);
            weight.x = exp2f(weight.x);
            weight.y = exp2f(weight.y);
            sums[i & 1] = add2(sums[i & 1], weight);
            words[part * 16 + i] = pack2<kFormat>(weight.x, weight.y);
          }
        }
        own = (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
        if (look == 4 || !__any_sync(0xffffffffu, own > kMostWeight)) break;
      }
      sum += own;
      tmem_st32(s_tmem, words);
      tmem_st32(s_tmem + 32, words + 32);
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kWeights0 + t));
    }
    // Output: a row's 256 bytes by its own thread, in whole sectors where rows begin with one.
    const int slot = kPieces ? walk.slot() : -1;
    const bool live = row < item.rows && slot == -1;
    if (p.lse != nullptr && live)
      p.lse[size_t(item.row + row) * p.heads + item.head] = sum > 0.f ? (reference + log2f(sum)) * 0.6931471805599453f : (sum == 0.f ? -INFINITY : sum);
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    char* out = static_cast<char*>(p.out) + (size_t(item.row + row) * p.heads + item.head) * (LATENT_NOPE * 2);
    if (steps > 0) {
      if (!warp_wait(sm.bar(kOut0 + t), outputs++ & 1, abort_flag)) return;
      tc_fence_after_sync();
    }
    if (kPieces && slot != -1) {
      if (slot == kNoPiece) continue;
      if (row < item.rows) p.statistics[size_t(slot) * kItemRows + row] = part_statistics(reference, sum);
      float* sums = p.sums + size_t(slot) * kSlotFloats + sums_place(row, 0);
#pragma unroll 1
      for (int c = 0; c < (steps > 0 ? kTile : 0); c += 32) {
        uint32_t o[32];
        tmem_ld32(o_tmem + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 8) store_sector(sums + (c + e) * 32, o + e);
      }
      tc_fence_before_sync();
      continue;
    }
#pragma unroll 1
    for (int c = 0; c < kTile; c += 32) {
      uint32_t o[32];
      if (steps > 0) {
        tmem_ld32(o_tmem + c, o);
        tmem_wait_ld();
      }
      uint32_t words[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        words[i] = sum == 0.f ? 0u : pack2<kFormat>(__uint_as_float(o[2 * i]) * inverse, __uint_as_float(o[2 * i + 1]) * inverse);
      if (live && p.sectors) {
        store_sector(out + c * 2, words);
        store_sector(out + c * 2 + 32, words + 8);
      } else if (live) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(out + c * 2 + i * 4) = make_uint4(words[i], words[i + 1], words[i + 2], words[i + 3]);
      }
    }
    tc_fence_before_sync();  // (the accumulator may be overwritten when this warp's next weights are there)
  }
}

template <int kFormat, bool kPieces>
__global__ void __launch_bounds__(kThreads, 1) prefill_kernel(const __grid_constant__ Params p) {
  extern __shared__ unsigned char smem_raw[];
  Shared sm;
  const uint32_t raw = smem_u32(smem_raw), pad = (1024u - (raw & 1023u)) & 1023u;
  sm.base = raw + pad;
  sm.ptr = smem_raw + pad;
  const int warp = threadIdx.x >> 5;
  wait_for_predecessor();
  let_successor_start();
  Item item;
  if (!find_item<kPieces>(p, blockIdx.x, item)) return;  // the whole block
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarCount; ++i)
      mbar_init(sm.bar(i), i >= kWeights0 && i < kWeights0 + 2 ? 4 : i >= kItemDone0 ? kSoftmaxWarps + 2 : 1);
    mbar_fence_init();
    *sm.abort_flag() = 0;
  }
  if (warp == kProductWarp) { tmem_alloc(smem_u32(sm.slot()), 512); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *sm.slot();
  // A softmax thread holds a row's 128 scores: the third warpgroup's registers go to the first two (200 + 200 + 104 of 3 x 168).
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n");
    softmax_role<kFormat, kPieces>(p, sm, tmem);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n");
    if (warp == kProductWarp) {
      if (elect_one()) {
        product_role<kFormat>(p, sm, tmem);
        if (*sm.abort_flag() != 0) wait_for_products(sm.bar(kGivenUp));
      }
      __syncwarp();
    } else if (warp == kCopyWarp) {
      copy_role(p, sm);
    } else if (warp == kPlanWarp) {
      plan_role<kPieces>(p, sm, item);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && *sm.abort_flag() != 0) report(p.status, SPARSE_MLA_STATUS_WAIT_EXPIRED, item.row, item.head);
  if (warp == kProductWarp) tmem_dealloc(tmem, 512);
}

// Items that were cut. Every block finds out what there is; 32 features of eight rows to one to eight of its warps. Bound by latency.
template <int kFormat>
__global__ void __launch_bounds__(kCombineThreads, 2) join_kernel(const __grid_constant__ Params p) {
  __shared__ Shares shared;
  wait_for_predecessor();
  let_successor_start();
  constexpr int kSegments = LATENT_NOPE / kUnitFeatures, kUnits = kItemRows / kUnitRows * kSegments;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Item item;
  Cut cut;
  if (!find_whole<true>(p, 0, item, &cut) || cut.pieces == 1) return;
  const int warps = warps_for(cut.pieces), turns = kUnits * warps / kCombineWarps;  // of a block for an item
  for (int turn = blockIdx.x;; turn += gridDim.x) {
    const int number = turn / turns;
    if (!find_whole<true>(p, number * cut.pieces, item, &cut)) return;  // the whole block
    const int count = cut.of(p, item);
    if (count == 1) continue;
    const int unit = ((turn - number * turns) * kCombineWarps + warp) / warps, segment = unit % kSegments;
    auto feature_of = [&](int lane) { return segment * kUnitFeatures + (lane >> 3) * 8; };
    join_parts<kFormat>(
        shared, warps, count, unit / kSegments * kUnitRows, item.rows,
        [&](int part, int row) { return p.sums + size_t(number * cut.pieces + part) * kSlotFloats + sums_place(row, feature_of(lane)); },
        [&](int part, int row) { return p.statistics + size_t(number * cut.pieces + part) * kItemRows + row; },
        [&](int row, int owner) { return static_cast<char*>(p.out) + ((size_t(item.row + row) * p.heads + item.head) * LATENT_NOPE + feature_of(owner)) * 2; },
        [&](int row, float reference, float sum, bool first_of_row) {
          if (p.lse != nullptr && first_of_row && segment == 0)
            p.lse[size_t(item.row + row) * p.heads + item.head] = sum > 0.f ? (reference + log2f(sum)) * 0.6931471805599453f : (sum == 0.f ? -INFINITY : sum);
          return sum == 0.f ? 0.f : 1.f / sum;
        });
  }
}

// The map of [rows, heads, features] with boxes of 128 rows of a head; *step: what a head adds to its coordinate (0: all share memory).
int map_heads(CUtensorMap* map, int format, const void* base, int64_t rows, int64_t heads, int64_t features, int64_t row_stride, int64_t head_stride, int32_t* step) {
  *step = heads > 1 && head_stride != 0;
  const int64_t sizes[3] = {features, *step ? heads : 1, rows};
  const int64_t strides[2] = {*step ? head_stride : features, rows > 1 ? row_stride : features};
  return encode_map(map, format, 3, base, sizes, strides, 2, kTile);
}

template <int kFormat, bool kPieces>
int launch(const Params& p, int blocks, cudaStream_t stream) {
  static bool configured[64] = {false};  // a per-device setting: plain words written with the same value by whoever gets there first
  int device = 0;
  if (const cudaError_t error = cudaGetDevice(&device)) return int(error);
  if (device < 0 || device >= 64) return -1;
  if (!configured[device]) {
    if (const cudaError_t error = cudaFuncSetAttribute(prefill_kernel<kFormat, kPieces>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes)) return int(error);
    configured[device] = true;
  }
  if (const cudaError_t error = launch_overlapped(prefill_kernel<kFormat, kPieces>, blocks, kThreads, kSmemBytes, stream, p)) return int(error);
  if constexpr (kPieces) return int(launch_overlapped(join_kernel<kFormat>, 2 * p.slots, kCombineThreads, 0, stream, p));
  return 0;
}

// Pieces that a call may be cut into: a block for every SM where even the most items that it may have take half of them, and requests may be long enough.
int slots_of(const latent_prefill_call& c) {
  const int64_t requests = c.tokens < c.batches ? c.tokens : c.batches;
  if (requests == 0 || c.keys <= (kLeastSteps + kSavedSteps - 1) * kTile) return 0;
  const int64_t items = requests + (c.tokens - requests) / kItemRows;  // of a head
  const int count = multiprocessors();
  return items * c.heads <= count / 2 ? count : 0;
}
inline size_t sums_offset(int slots) { return size_t(slots) * kItemRows * sizeof(float2); }

}  // namespace prefill
}  // namespace latent

extern "C" int workspace_size_latent_prefill(uint64_t* bytes, const latent_prefill_call* call) {
  using namespace latent;
  if (bytes == nullptr || call == nullptr || call->tokens < 0 || call->batches < 0 || call->keys < 0 || call->heads < 0 || call->heads > 65535) return -1;
  const int slots = prefill::slots_of(*call);
  *bytes = prefill::sums_offset(slots) + size_t(slots) * prefill::kSlotFloats * sizeof(float);
  return 0;
}

extern "C" int launch_latent_prefill(void* stream, const latent_prefill_call* call) {
  using namespace latent;
  if (call == nullptr) return -1;
  const latent_prefill_call& c = *call;
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || !scale_fits(c.scale) || c.status == nullptr) return -1;
  if (c.batches < 0 || c.batches >= INT32_MAX || c.tokens < 0 || c.tokens > INT32_MAX - 256 || c.keys < 0 || c.keys > INT32_MAX - 256 || c.heads < 1 || c.heads > 65535) return -1;
  int64_t blocks = (c.tokens / 256 + c.batches) * c.heads;  // at least as many as there are items
  if (blocks > INT32_MAX) return -1;
  // (what has no entries has no alignment)
  if (c.tokens > 0 && (!aligned(c.q) || !aligned(c.out) || (c.q_token | c.q_head) % 8 != 0)) return -1;
  if (c.keys > 0 && (!aligned(c.k) || !aligned(c.v) || !aligned(c.k_rope) || (c.k_token | c.k_head | c.v_token | c.v_head | c.rope_token) % 8 != 0)) return -1;
  if (c.tokens == 0 || c.batches == 0) return 0;
  prefill::Params p = {};
  p.slots = prefill::slots_of(c);
  if (p.slots > 0) {
    if (c.workspace == nullptr || reinterpret_cast<uintptr_t>(c.workspace) % 32 != 0) return -1;
    p.statistics = static_cast<float2*>(c.workspace);
    p.sums = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + prefill::sums_offset(p.slots));
    if (blocks < p.slots) blocks = p.slots;
  }
  const int64_t keys = c.keys > 0 ? c.keys : 1;  // (without keys nothing is copied)
  const void* any = c.q;
  if (const int e = prefill::map_heads(&p.q, c.type, c.q, c.tokens, c.heads, prefill::kFeatures, c.q_token, c.q_head, &p.q_head)) return e;
  if (const int e = prefill::map_heads(&p.k, c.type, c.keys > 0 ? c.k : any, keys, c.keys > 0 ? c.heads : 1, LATENT_NOPE, c.k_token, c.k_head, &p.k_head)) return e;
  if (const int e = prefill::map_heads(&p.v, c.type, c.keys > 0 ? c.v : any, keys, c.keys > 0 ? c.heads : 1, LATENT_NOPE, c.v_token, c.v_head, &p.v_head)) return e;
  const int64_t sizes[2] = {LATENT_ROPE, keys}, strides[1] = {keys > 1 ? c.rope_token : LATENT_ROPE};
  if (const int e = sm100::encode_map(&p.rope, c.type, 2, c.keys > 0 ? c.k_rope : any, sizes, strides, 1, prefill::kTile)) return e;
  p.cu_q = c.cu_seqlens_q;
  p.cu_k = c.cu_seqlens_k;
  p.out = c.out;
  p.lse = c.lse;
  p.status = c.status;
  p.batches = int32_t(c.batches);
  p.tokens = int32_t(c.tokens);
  p.keys = int32_t(c.keys);
  p.heads = int32_t(c.heads);
  p.causal = c.causal;
  p.sectors = reinterpret_cast<uintptr_t>(c.out) % 32 == 0;
  p.scale_log2 = float(c.scale * 1.4426950408889634);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.slots > 0) return c.type == LATENT_BF16 ? prefill::launch<1, true>(p, int(blocks), s) : prefill::launch<0, true>(p, int(blocks), s);
  return c.type == LATENT_BF16 ? prefill::launch<1, false>(p, int(blocks), s) : prefill::launch<0, false>(p, int(blocks), s);
}
