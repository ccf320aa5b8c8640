// The plan of the absorbed attention call on the CPU: `plan_block` and `plan_role`, taken from the kernel's source (plan.inc), with a fiber for every
// thread of a block. stdin, 32-bit words: blocks, heads, requests, pages, page rows, tokens, then cu_seqlens_q and seqused_kv. stdout: for each
// block, its pieces (row, rows, request, token, head, base, length, first, last, slot; first -1 behind the last) and its record (row, rows, head, last, and
// whether slot 2 i is said to be empty).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <vector>
#include <ucontext.h>

#define __device__
#define __forceinline__ inline
#define LATENT_VALUES 512
using std::max;
using std::min;
struct float2 { float x, y; };
inline float2 make_float2(float x, float y) { return {x, y}; }
using CUtensorMap = int;
struct Index { unsigned x; } threadIdx, blockIdx, gridDim;
template <typename T> inline T __ldg(const T* at) { return *at; }
inline int __ffs(unsigned v) { return __builtin_ffs(int(v)); }

// ---- the block's threads ------------------------------------------------------------------------
struct Meeting { int64_t value[2][32]; int arrived; unsigned generation; } warps[16];
constexpr int kBlockThreads = 512;
int running, block_arrived;
unsigned block_generation;
ucontext_t scheduler, fibers[kBlockThreads];
std::vector<char> stacks(kBlockThreads * size_t(65536));
bool finished[kBlockThreads];
std::function<void()> body;

inline void yield() {
  const unsigned thread = threadIdx.x;
  swapcontext(&fibers[thread], &scheduler);
  threadIdx.x = thread;
}
void enter() {
  body();
  finished[threadIdx.x] = true;
  if (block_arrived == --running && block_arrived > 0) { block_arrived = 0; ++block_generation; }
  swapcontext(&fibers[threadIdx.x], &scheduler);
}
inline void __syncthreads() {
  const unsigned generation = block_generation;
  if (++block_arrived == running) { block_arrived = 0; ++block_generation; }
  while (block_generation == generation) yield();
}
inline const int64_t* meet(int64_t mine) {
  Meeting& warp = warps[threadIdx.x >> 5];
  const unsigned generation = warp.generation;
  warp.value[generation & 1][threadIdx.x & 31] = mine;
  if (++warp.arrived == 32) { warp.arrived = 0; ++warp.generation; }
  while (warp.generation == generation) yield();
  return warp.value[generation & 1];
}
template <typename T> inline T __shfl_up_sync(unsigned, T v, int d) { const int lane = threadIdx.x & 31; return T(meet(v)[lane >= d ? lane - d : lane]); }
template <typename T> inline T __shfl_sync(unsigned, T v, int from) { return T(meet(v)[from]); }
template <typename T> inline T __shfl_xor_sync(unsigned, T v, int d) { const int lane = threadIdx.x & 31; return T(meet(v)[lane ^ d]); }
inline unsigned __ballot_sync(unsigned, bool v) {
  const int64_t* all = meet(v);
  unsigned mask = 0;
  for (int i = 0; i < 32; ++i) mask |= unsigned(all[i] != 0) << i;
  return mask;
}
inline int __reduce_max_sync(unsigned, int v) { const int64_t* all = meet(v); return int(*std::max_element(all, all + 32)); }
inline int __reduce_min_sync(unsigned, int v) { const int64_t* all = meet(v); return int(*std::min_element(all, all + 32)); }
template <typename T> inline T __reduce_add_sync(unsigned, T v) { const int64_t* all = meet(v); T sum = 0; for (int i = 0; i < 32; ++i) sum += T(all[i]); return sum; }
inline bool run_block() {
  running = kBlockThreads;
  block_arrived = 0;
  memset(warps, 0, sizeof(warps));
  for (int t = 0; t < kBlockThreads; ++t) {
    finished[t] = false;
    getcontext(&fibers[t]);
    fibers[t].uc_stack.ss_sp = &stacks[t * size_t(65536)];
    fibers[t].uc_stack.ss_size = 65536;
    fibers[t].uc_link = nullptr;
    makecontext(&fibers[t], enter, 0);
  }
  for (int round = 0; round < 1000000; ++round) {
    bool left = false;
    for (int t = 0; t < kBlockThreads; ++t)
      if (!finished[t]) { threadIdx.x = t; swapcontext(&scheduler, &fibers[t]); left = true; }
    if (!left) return true;
  }
  return false;
}

// ---- what the plan announces ----------------------------------------------------------------------
void announced_on(uint32_t bar);
inline void mbar_arrive(uint32_t bar) { announced_on(bar); }
struct Shared;
constexpr long long kLongWait = 1ll << 36;
inline bool warp_wait(uint32_t, uint32_t, volatile int*, long long) { meet(0); return true; }

#include "plan.inc"

std::vector<Piece> pieces;
const Shared* current;
void announced_on(uint32_t bar) { pieces.push_back(*current->piece((bar / 8 - kPieceReady0) % kPieces)); }

int main() {
  int32_t head[6];
  if (fread(head, 4, 6, stdin) != 6) return 1;
  const int blocks = head[0], batches = head[2];
  std::vector<int32_t> cu(batches + 1), lengths(batches);
  if (int(fread(cu.data(), 4, batches + 1, stdin)) != batches + 1 || int(fread(lengths.data(), 4, batches, stdin)) != batches) return 1;
  Params p = {};
  p.heads = head[1];
  p.by_heads = divisor_of(p.heads);
  p.tile_tokens = kRows / p.heads + 1;
  p.batches = batches;
  p.pages = head[3];
  p.page_rows = head[4];
  p.tokens = head[5];
  p.cu = cu.data();
  p.lengths = lengths.data();
  std::vector<Record> records(blocks);
  std::vector<float2> statistics(size_t(blocks) * 2 * kRows);
  p.records = records.data();
  p.statistics = statistics.data();
  gridDim.x = blocks;
  std::vector<unsigned char> memory(4096);
  for (int block = 0; block < blocks; ++block) {
    blockIdx.x = block;
    Shared sm = {};
    sm.ptr = memory.data();
    sm.bars = 0;
    sm.pieces = 2048;
    sm.misc = 3328;
    current = &sm;
    pieces.clear();
    statistics[size_t(2 * block) * kRows] = {1.f, 1.f};
    body = [&] {
      Place place = {};
      Borders borders = {};
      if (batches > 32) {
        borders = plan_block<kBlockThreads / 32>(p, reinterpret_cast<int64_t*>(memory.data()), &place);
        __syncthreads();
      }
      if (threadIdx.x >> 5 != kPlanWarp) return;
      if (batches <= 32) borders = plan_block<1>(p, nullptr, &place);
      plan_role(p, sm, borders, place);
    };
    if (!run_block()) { fprintf(stderr, "block %d: somebody waits for ever\n", block); return 2; }
    for (const Piece& q : pieces) {
      const int64_t words[10] = {q.row, q.rows, q.request, q.token, q.head, q.base, q.length, q.first, q.last, q.slot};
      fwrite(words, 8, 10, stdout);
    }
    const Record& r = records[block];
    const int64_t words[5] = {r.row, r.rows, r.head, r.last, statistics[size_t(2 * block) * kRows].x != 1.f};
    fwrite(words, 8, 5, stdout);
  }
  return 0;
}
