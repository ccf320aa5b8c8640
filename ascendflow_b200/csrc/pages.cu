// The pages of a cache: who has which, on the device and without waiting (a step that grows requests may be captured in a graph).
//
// All three operators rank things in a fixed order: free pages by number, wishes by request and entry. One cluster of eight blocks does that: a
// block marks the pages of its eighth as bits in shared memory, the blocks exchange their sums, and each knows what is in front of it; the cluster's barrier costs a
// fraction of a microsecond where another launch costs two. Pages are copied by a second kernel on all SMs, which also writes what is long and needs no order (a fork's
// table, a compacted one). Resizing a large table is shared out in the same way: what eight SMs read of it would take longer than two more launches.
//
// Bound by latency (chains of loads, and four cluster barriers) for small tables, by memory for copies.
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/pages.h"
#include "../../include/sparse_mla.h"
#include "latent_common.cuh"

namespace pages {
namespace {

using namespace sm100;
using latent::report;

constexpr int kCluster = 8, kThreads = 1024, kWarps = kThreads / 32;

struct Plan {
  pages_call c;
  const int32_t* parents;
  int32_t* places;
  int32_t children;
  int32_t *numbers;            // free pages in order; compact: the pages that are moved
  int32_t *first, *heirs;      // resize: a request's first entry that wishes, its number of wishes; fork: its first child, its number of children
  int32_t *ranks;              // resize: wishes in front of a request's; fork: the page that a child has of its own, -1: none was left, kShared
  int32_t *free;               // pages in `numbers`
  uint32_t *marks;             // [8 words] of all blocks, where they have been made in front
  int4* copies;                // source, target, rows
  int32_t* copy_count;
  int32_t words;               // of 32 pages, per block
};

constexpr int kShared = -2;

struct Shared {
  int32_t totals[4][kCluster];  // what the blocks tell each other
  int32_t sums[kWarps];
  uint32_t marks[1];            // [words]
};

__device__ __forceinline__ void meet() {
  cluster_arrive();
  cluster_wait();
}
// Tells all blocks of the cluster this block's `value`; read behind the next meeting. One thread for each of them. (The first time behind a meeting: they have to run.)
__device__ __forceinline__ void tell(Shared& sm, int which, int rank, int value) {
  if (threadIdx.x < kCluster) {
    const uint32_t at = cluster_address(smem_u32(&sm.totals[which][rank]), threadIdx.x);
    asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(at), "r"(value) : "memory");
  }
}
__device__ __forceinline__ int in_front(const Shared& sm, int which, int rank) {
  int sum = 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) sum += r < rank ? sm.totals[which][r] : 0;
  return sum;
}
__device__ __forceinline__ int in_all(const Shared& sm, int which) { return in_front(sm, which, kCluster); }

// Sum over the block, for all threads.
__device__ __forceinline__ int block_sum(Shared& sm, int value) {
  value = __reduce_add_sync(0xffffffffu, value);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm.sums[threadIdx.x >> 5] = value;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, sm.sums[threadIdx.x & 31]);
}
// Sum over the threads in front; *total over all.
__device__ __forceinline__ int block_rank(Shared& sm, int value, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inclusive = value;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, inclusive, d);
    if (lane >= d) inclusive += other;
  }
  __syncthreads();
  if (lane == 31) sm.sums[warp] = inclusive;
  __syncthreads();
  const int sum = sm.sums[lane];
  *total = __reduce_add_sync(0xffffffffu, sum);
  return inclusive - value + __reduce_add_sync(0xffffffffu, lane < warp ? sum : 0);
}

// Marks of this block's pages: bit i of word w for page 32 (rank * words + w) + i. Free pages (kUsed: those in use); their number. Copies the counts where there are two.
template <bool kUsed>
__device__ __forceinline__ int mark_pages(const Plan& p, Shared& sm, int rank, const int32_t* counts, int32_t* copy) {
  const int lane = threadIdx.x & 31, warp = kWarps - 1 - (threadIdx.x >> 5), blocks = int(p.c.blocks);  // (the first warps may have more to do)
  constexpr int kInFlight = 8;
  int found = 0;
  for (int word = warp; word < p.words; word += kWarps * kInFlight) {
    int count[kInFlight];
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) {
      const int64_t page = int64_t(rank * p.words + word + n * kWarps) * 32 + lane;
      count[n] = word + n * kWarps < p.words && page < blocks ? __ldcg(counts + page) : INT_MIN;
    }
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) {
      const uint32_t marks = __ballot_sync(0xffffffffu, kUsed ? count[n] != INT_MIN && count[n] != 0 : count[n] == 0);
      if (word + n * kWarps < p.words) {
        if (lane == 0) sm.marks[word + n * kWarps] = marks;
        const int64_t page = int64_t(rank * p.words + word + n * kWarps) * 32 + lane;
        if (copy != nullptr && page < blocks) copy[page] = count[n];
        found += __popc(marks);
      }
    }
  }
  return block_sum(sm, lane == 0 ? found : 0);
}

// The same of marks that have been made.
__device__ __forceinline__ int fetch_marks(const Plan& p, Shared& sm, int rank) {
  constexpr int kInFlight = 4;
  int found = 0;
  for (int word = threadIdx.x; word < p.words; word += kThreads * kInFlight) {
    uint32_t marks[kInFlight];
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) marks[n] = word + n * kThreads < p.words ? p.marks[rank * p.words + word + n * kThreads] : 0;
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) {
      if (word + n * kThreads < p.words) sm.marks[word + n * kThreads] = marks[n];
      found += __popc(marks[n]);
    }
  }
  return block_sum(sm, found);
}

// Calls list(rank, page) for the marked pages of this block (behind a filter of words), ranks from `rank` on; stops at `most`. A warp goes through its words one by one, a
// page to a lane, so that what is listed is stored side by side, or, where there are fewer marks in each word than such words, a word to a
// lane; with room for them (`staged`), up to kStaged of a warp's pages go through shared memory instead
// (a large table's: 73 K pages, seven to a word, are listed in 10 us by either of the others, and in 4 so).
constexpr int kStaged = 512;
template <class Filter, class List>
__device__ __forceinline__ void list_marked(const Plan& p, Shared& sm, int block_rank_, int rank, int most, Filter filter, List list, uint16_t (*staged)[kStaged] = nullptr) {
  for (int word0 = 0; word0 < p.words && rank < most; word0 += kThreads) {
    const int word = word0 + int(threadIdx.x);
    const int page0 = (block_rank_ * p.words + word) * 32, lane = threadIdx.x & 31;
    const uint32_t marks = word < p.words ? filter(sm.marks[word], page0) : 0u;
    int total, own = rank + block_rank(sm, __popc(marks), &total);
    uint32_t left = __ballot_sync(0xffffffffu, marks != 0 && own < most);
    if (const int all = __reduce_add_sync(0xffffffffu, __popc(marks)); staged != nullptr && all <= kStaged) {
      const int first = __shfl_sync(0xffffffffu, own, 0), page_of_warp = __shfl_sync(0xffffffffu, page0, 0);
      uint16_t* const found = staged[threadIdx.x >> 5];
      int at = own - first;
      for (uint32_t mine = marks; mine != 0; mine &= mine - 1) found[at++] = uint16_t(lane * 32 + __ffs(mine) - 1);
      __syncwarp();
      for (int i = lane; i < min(all, most - first); i += 32) list(first + i, page_of_warp + found[i]);
      __syncwarp();
      left = 0;
    } else if (int(__reduce_max_sync(0xffffffffu, uint32_t(__popc(marks)))) < __popc(left)) {
      for (uint32_t mine = marks; mine != 0 && own < most; mine &= mine - 1, ++own) list(own, page0 + __ffs(mine) - 1);
      left = 0;
    }
    for (; left != 0; left &= left - 1) {
      const int from = __ffs(left) - 1, page = __shfl_sync(0xffffffffu, page0, from) + lane;
      const uint32_t theirs = __shfl_sync(0xffffffffu, marks, from);
      const int place = __shfl_sync(0xffffffffu, own, from) + __popc(theirs & ((1u << lane) - 1u));
      if ((theirs >> lane & 1) && place < most) list(place, page);
    }
    rank += total;
  }
}

// Bits of pages below `border` in the word that begins with `page0`.
__device__ __forceinline__ uint32_t below(int page0, int border) {
  const int n = min(max(border - page0, 0), 32);
  return n == 32 ? 0xffffffffu : (1u << n) - 1u;
}

// What a length counts: rows (within the table) and entries.
struct Extent {
  int64_t rows;
  int entries;
};
__device__ __forceinline__ Extent extent_of(const Plan& p, int request, int length, bool reports) {
  const int64_t room = p.c.entries * p.c.page_rows;
  if (reports && length > room) report(p.c.status, SPARSE_MLA_STATUS_BAD_PAGE, request, length);
  const int64_t rows = min(int64_t(max(length, 0)), room);
  return {rows, int((rows + p.c.page_rows - 1) / p.c.page_rows)};
}
__device__ __forceinline__ bool names_page(const Plan& p, int entry) { return unsigned(entry) < unsigned(p.c.blocks); }

// Calls each(i, entry) for a thread's share of `entries` entries, several loads at a time.
template <class Each>
__device__ __forceinline__ void each_entry(const int32_t* row, int entries, int thread, int threads, Each each) {
  constexpr int kInFlight = 8;
  for (int at = thread; at < entries; at += threads * kInFlight) {
    int entry[kInFlight];
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) entry[n] = at + threads * n < entries ? row[at + threads * n] : -1;
#pragma unroll
    for (int n = 0; n < kInFlight; ++n)
      if (at + threads * n < entries) each(at + threads * n, entry[n]);
  }
}

// ---- resize ---------------------------------------------------------------------------------------------------------

// Counts to another tensor, several at a time.
__device__ __forceinline__ void copy_counts(const Plan& p, int64_t thread, int64_t threads) {
  constexpr int kInFlight = 8;
  for (int64_t at = thread; at < p.c.blocks; at += threads * kInFlight) {
    int count[kInFlight];
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) count[n] = at + n * threads < p.c.blocks ? p.c.counts_in[at + n * threads] : 0;
#pragma unroll
    for (int n = 0; n < kInFlight; ++n)
      if (at + n * threads < p.c.blocks) p.c.counts_out[at + n * threads] = count[n];
  }
}

// What a request gives back, and what it keeps; entry by entry, by `threads` threads. Wishes of this thread's entries, the first of them.
__device__ __forceinline__ int release(const Plan& p, int request, int thread, int threads, int* first) {
  const Extent extent = extent_of(p, request, p.c.lengths[request], thread == 0);
  const int entries = int(p.c.entries);
  const int32_t* in = p.c.table_in + int64_t(request) * entries;
  int32_t* out = p.c.table_out + int64_t(request) * entries;
  int own = 0;
  *first = INT_MAX;
  each_entry(in, entries, thread, threads, [&](int i, int entry) {
    const bool has = names_page(p, entry), counts = i < extent.entries;
    if (has && !counts) atomicSub(p.c.counts_out + entry, 1);
    if (!has && counts) {
      ++own;
      *first = min(*first, i);
    }
    const int next = has && counts ? entry : -1;
    if (in != out || next != entry) out[i] = next;
  });
  return own;
}

// A request's wishes, `wishes` from entry `first` on, get the free pages from rank `rank` on.
__device__ __forceinline__ void give(const Plan& p, int request, int thread, int threads, int rank, int wishes, int first, int free) {
  int32_t* out = p.c.table_out + int64_t(request) * p.c.entries;
  auto take = [&](int i, int place) {
    if (place < free) {
      const int page = __ldcg(p.numbers + place);
      out[i] = page;
      p.c.counts_out[page] = 1;
    } else {
      report(p.c.status, SPARSE_MLA_STATUS_NO_PAGE, request, i);
    }
  };
  const int counted = extent_of(p, request, p.c.lengths[request], false).entries;
  if (counted - first == wishes) {  // one after the other, as where a request has grown
    for (int i = thread; i < wishes; i += threads) take(first + i, rank + i);
  } else if (thread < 32) {
    for (int i0 = first; i0 < counted; i0 += 32) {
      const int i = i0 + thread;
      const bool wants = i < counted && out[i] < 0;
      const unsigned wanting = __ballot_sync(0xffffffffu, wants);
      if (wants) take(i, rank + __popc(wanting & ((1u << thread) - 1u)));
      rank += __popc(wanting);
    }
  }
}

// The list of the free pages, which are marked; the requests' ranks. By the cluster. The blocks' wishes are in totals[0] behind the next meeting.
__device__ __forceinline__ void rank_wishes(const Plan& p, Shared& sm, int rank, int begin, int end, int free_here, uint16_t (*staged)[kStaged] = nullptr) {
  tell(sm, 1, rank, free_here);
  meet();
  list_marked(p, sm, rank, in_front(sm, 1, rank), in_all(sm, 0), [](uint32_t marks, int) { return marks; }, [&](int at, int page) { p.numbers[at] = page; }, staged);
  int rank_of_tile = in_front(sm, 0, rank);
  for (int tile = begin; tile < end; tile += kThreads) {
    const int request = tile + int(threadIdx.x), own = request < end ? p.heirs[request] : 0;
    int total;
    const int start = rank_of_tile + block_rank(sm, own, &total);
    if (request < end) p.ranks[request] = start;
    rank_of_tile += total;
  }
}

// The whole of it, for a small table.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 1) resize_kernel(const __grid_constant__ Plan p) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  const int rank = int(cluster_rank()), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, requests = int(p.c.requests);
  const int share = (requests + kCluster - 1) / kCluster, begin = min(rank * share, requests), end = min(begin + share, requests);
  wait_for_predecessor();
  let_successor_start();
  if (p.c.counts_in != p.c.counts_out) copy_counts(p, rank * kThreads + threadIdx.x, kCluster * kThreads);
  meet();
  int wishes = 0;
  for (int request = begin + warp; request < end; request += kWarps) {
    int first, own = release(p, request, lane, 32, &first);
    own = __reduce_add_sync(0xffffffffu, own);
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) {
      p.first[request] = first;
      p.heirs[request] = own;
    }
    wishes += own;
  }
  wishes = block_sum(sm, lane == 0 ? wishes : 0);
  tell(sm, 0, rank, wishes);
  meet();
  rank_wishes(p, sm, rank, begin, end, mark_pages<false>(p, sm, rank, p.c.counts_out, nullptr));
  meet();  // (the last: nobody is told anything behind it)
  const int free = in_all(sm, 1);
  for (int request = begin + warp; request < end; request += kWarps) {
    const int own = p.heirs[request];
    if (own > 0) give(p, request, lane, 32, p.ranks[request], own, p.first[request], free);
  }
}

// A large table, or long rows: a block to each request in front and behind, the cluster between. By the cluster alone / so, called eagerly, us (in brackets replayed from a graph): 128 requests of
// 129 entries 9.7 / 13.1 (9.6 / 10.1), 64 of 513 10.8 / 13.5 (10.4 / 10.5), 128 of 513 12.7 / 13.3 (12.3 / 11.3), 512 of 129 14.3 / 13.7, 1024 of 129 20.8 / 16.3; 1024 of 2049, 700 K pages 192 / 24. A warp goes
// through a row alone: 16 rows of 1025 11.1 / 13.2, one of 2049 13.0 / 13.0, 4 of 8193 28.0 / 14.5, one of 32769 84 / 23.
constexpr int kRowThreads = 256;
constexpr int64_t kSmallTable = 1 << 16, kShortRow = 1 << 11;

__global__ void __launch_bounds__(kRowThreads) copy_counts_kernel(const __grid_constant__ Plan p) {
  wait_for_predecessor();
  let_successor_start();
  copy_counts(p, int64_t(blockIdx.x) * kRowThreads + threadIdx.x, int64_t(gridDim.x) * kRowThreads);
}

__global__ void __launch_bounds__(kRowThreads) release_kernel(const __grid_constant__ Plan p) {
  __shared__ int counts[kRowThreads / 32], firsts[kRowThreads / 32];
  wait_for_predecessor();
  let_successor_start();
  const int request = blockIdx.x;
  int first, own = release(p, request, threadIdx.x, kRowThreads, &first);
  own = __reduce_add_sync(0xffffffffu, own);
  first = __reduce_min_sync(0xffffffffu, first);
  if ((threadIdx.x & 31) == 0) {
    counts[threadIdx.x >> 5] = own;
    firsts[threadIdx.x >> 5] = first;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kRowThreads / 32; ++w) {
      own += counts[w];
      first = min(first, firsts[w]);
    }
    p.first[request] = first;
    p.heirs[request] = own;
  }
}

// Marks of all pages, eight words by a warp, where there are many. Without / with, called eagerly, us (in brackets replayed from a graph), 256 requests with 256 to 10 K wishes: 80 K pages
// 14.2-15.8 / 15.4-16.0 (12.6-14.3 / 12.0-13.7), 131 K 14.7-18.5 / 15.5-17.3 (12.9-16.6 / 12.0-15.7), 200 K 16.8-21.2 / 16.2-18.2 (15.1-19.6 / 12.2-16.7), 262 K 17.5-21.5 / 15.5-17.8, 700 K
// 27.4-31.5 / 15.5-19.6.
constexpr int kWordsPerWarp = 8, kManyPages = 1 << 17;
__global__ void __launch_bounds__(kRowThreads) mark_kernel(const __grid_constant__ Plan p) {
  wait_for_predecessor();
  let_successor_start();
  const int lane = threadIdx.x & 31, first = (int(blockIdx.x) * (kRowThreads / 32) + int(threadIdx.x >> 5)) * kWordsPerWarp;
  int count[kWordsPerWarp];
#pragma unroll
  for (int n = 0; n < kWordsPerWarp; ++n) count[n] = (first + n) * 32 + lane < int(p.c.blocks) ? p.c.counts_out[(first + n) * 32 + lane] : 1;
#pragma unroll
  for (int n = 0; n < kWordsPerWarp; ++n) {
    const uint32_t marks = __ballot_sync(0xffffffffu, count[n] == 0);
    if (lane == n && first + n < kCluster * p.words) p.marks[first + n] = marks;
  }
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 1) rank_kernel(const __grid_constant__ Plan p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint16_t staged[kWarps][kStaged];
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  const int rank = int(cluster_rank()), requests = int(p.c.requests);
  const int share = (requests + kCluster - 1) / kCluster, begin = min(rank * share, requests), end = min(begin + share, requests);
  wait_for_predecessor();
  let_successor_start();
  cluster_arrive_relaxed();
  int wishes = 0;
  for (int request = begin + int(threadIdx.x); request < end; request += kThreads) wishes += p.heirs[request];
  wishes = block_sum(sm, wishes);
  const int free_here = p.marks != nullptr ? fetch_marks(p, sm, rank) : mark_pages<false>(p, sm, rank, p.c.counts_out, nullptr);
  cluster_wait();  // (all blocks run)
  tell(sm, 0, rank, wishes);
  rank_wishes(p, sm, rank, begin, end, free_here, staged);
  if (rank == 0 && threadIdx.x == 0) *p.free = in_all(sm, 1);
  meet();  // (nobody leaves while others are told)
}

__global__ void __launch_bounds__(kRowThreads) give_kernel(const __grid_constant__ Plan p) {
  wait_for_predecessor();
  let_successor_start();
  const int request = blockIdx.x, own = p.heirs[request];
  if (own > 0) give(p, request, threadIdx.x, kRowThreads, p.ranks[request], own, p.first[request], *p.free);
}

// ---- copies ---------------------------------------------------------------------------------------------------------

constexpr int kCopyThreads = 256, kUnitBytes = 16384, kCopyBlocks = 5;  // per SM

struct Copies {
  Plan plan;
  bool forks;
  int64_t entries;  // of a table that gets new numbers
  int64_t page_rows;
  int32_t tensors, units;  // units of all tensors, for one copy
  struct {
    char* memory;
    int64_t page_bytes;
    int32_t rows, first_unit;
  } tensor[PAGES_MOST_TENSORS];
};

__device__ __forceinline__ uint4 load_once(const uint4* at) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at) : "memory");
  return v;
}

// Row `child` of the new table.
__device__ __forceinline__ void write_row(const Plan& p, int child, int thread, int threads) {
  const int entries = int(p.c.entries), parent = p.parents[child], last_page = __ldcg(p.ranks + child);
  const int counted = unsigned(parent) < unsigned(p.c.requests) ? extent_of(p, parent, p.c.lengths[parent], false).entries : 0;
  int32_t* out = p.c.table_out + int64_t(child) * entries;
  if (counted > 0)
    each_entry(p.c.table_in + int64_t(parent) * entries, counted, thread, threads, [&](int i, int entry) {
      if (i == counted - 1 && last_page != kShared) entry = last_page;
      out[i] = names_page(p, entry) ? entry : -1;
    });
  for (int i = counted + thread; i < entries; i += threads) out[i] = -1;
}

// A request's entries as they were: one reference less, and one more for each row that has them. (Other pages than those that are given out.)
__device__ __forceinline__ void count_entries(const Plan& p, int request, int thread, int threads) {
  const int entries = int(p.c.entries);
  const Extent extent = extent_of(p, request, p.c.lengths[request], thread == 0);
  const int heirs = __ldcg(p.heirs + request), filled = int(extent.rows % p.c.page_rows);
  const int keeps = heirs > 0 && __ldcg(p.ranks + __ldcg(p.first + request)) == kShared;  // its first child, the last page
  each_entry(p.c.table_in + int64_t(request) * entries, entries, thread, threads, [&](int i, int page) {
    const int more = (i >= extent.entries ? 0 : i == extent.entries - 1 && filled != 0 ? keeps : heirs) - 1;
    if (more != 0 && names_page(p, page)) atomicAdd(p.c.counts_out + page, more);
  });
}

// What there is to do besides the plan: a fork's rows and counts, a compacted table's numbers; copies. By `workers` times kCopyThreads threads. 16 KiB of a page go at a time, 64 bytes by a
// thread with all loads in flight; what is not 16-byte aligned byte by byte (scales of a few bytes).
__device__ __forceinline__ void write_and_copy(const Copies& all, int worker, int workers, int thread) {
  const Plan& plan = all.plan;
  if (all.forks) {
    for (int child = worker; child < plan.children; child += workers) write_row(plan, child, thread, kCopyThreads);
    for (int request = worker; request < int(plan.c.requests); request += workers) count_entries(plan, request, thread, kCopyThreads);
  }
  for (int64_t i = int64_t(worker) * kCopyThreads + thread; i < all.entries; i += int64_t(workers) * kCopyThreads) {
    const int page = plan.c.table_in[i];
    plan.c.table_out[i] = names_page(plan, page) ? __ldcg(plan.places + page) : page;
  }
  const int64_t items = int64_t(__ldcg(plan.copy_count)) * all.units;
  for (int64_t item = worker; item < items; item += workers) {
    const int which = int(item / all.units), unit = int(item - int64_t(which) * all.units);
    int tensor = 0;
    for (int high = all.tensors; high - tensor > 1;) {
      const int middle = (tensor + high) >> 1;
      if (all.tensor[middle].first_unit <= unit) tensor = middle; else high = middle;
    }
    const int4 copy = __ldcg(plan.copies + which);
    const int64_t page_bytes = all.tensor[tensor].page_bytes, rows = all.tensor[tensor].rows;
    const int64_t first = int64_t(unit - all.tensor[tensor].first_unit) * kUnitBytes;
    const int64_t filled = (copy.z * rows + all.page_rows - 1) / all.page_rows * (page_bytes / rows);  // bytes of the page to copy
    const int bytes = int(min(filled - first, int64_t(kUnitBytes)));
    if (bytes <= 0) continue;
    const char* source = all.tensor[tensor].memory + copy.x * page_bytes + first;
    char* target = all.tensor[tensor].memory + copy.y * page_bytes + first;
    int done = 0;
    if (((reinterpret_cast<uintptr_t>(source) | reinterpret_cast<uintptr_t>(target)) & 15) == 0) {
      const int words = bytes / 16;
      uint4 v[kUnitBytes / 16 / kCopyThreads];
#pragma unroll
      for (int n = 0; n < kUnitBytes / 16 / kCopyThreads; ++n) {
        const int at = n * kCopyThreads + thread;
        if (at < words) v[n] = load_once(reinterpret_cast<const uint4*>(source) + at);
      }
#pragma unroll
      for (int n = 0; n < kUnitBytes / 16 / kCopyThreads; ++n) {
        const int at = n * kCopyThreads + thread;
        if (at < words) reinterpret_cast<uint4*>(target)[at] = v[n];
      }
      done = words * 16;
    }
    for (int at = done + thread; at < bytes; at += kCopyThreads) target[at] = source[at];
  }
}

__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) copy_kernel(const __grid_constant__ Copies all) {
  wait_for_predecessor();
  let_successor_start();
  write_and_copy(all, blockIdx.x, gridDim.x, threadIdx.x);
}

// The same at the end of a plan, by its blocks.
__device__ __forceinline__ void write_and_copy_here(const Copies& all, int rank) {
  meet();
  write_and_copy(all, rank * (kThreads / kCopyThreads) + int(threadIdx.x) / kCopyThreads, kCluster * (kThreads / kCopyThreads), int(threadIdx.x) % kCopyThreads);
}

// ---- fork -----------------------------------------------------------------------------------------------------------

template <bool kCopies>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 1) fork_kernel(const __grid_constant__ Copies all) {
  const Plan& p = all.plan;
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  const int rank = int(cluster_rank());
  const int requests = int(p.c.requests), entries = int(p.c.entries), children = p.children;
  const int share = (children + kCluster - 1) / kCluster, begin = min(rank * share, children), end = min(begin + share, children);
  wait_for_predecessor();
  let_successor_start();
  for (int request = rank * kThreads + threadIdx.x; request < requests; request += kCluster * kThreads) {
    p.first[request] = INT_MAX;
    p.heirs[request] = 0;
  }
  cluster_arrive();
  struct Tail {
    int parent;      // or -1
    int page, rows;  // the partly filled page, or -1, and its rows
    int count;       // of entries that name it
  };
  auto tail_of = [&](int child) {
    Tail tail = {p.parents[child], -1, 0, 0};
    if (unsigned(tail.parent) >= unsigned(requests)) tail.parent = -1;
    if (tail.parent < 0) return tail;
    const Extent extent = extent_of(p, tail.parent, p.c.lengths[tail.parent], false);
    tail.rows = int(extent.rows % p.c.page_rows);
    if (tail.rows == 0) return tail;
    const int page = p.c.table_in[int64_t(tail.parent) * entries + extent.entries - 1];
    if (!names_page(p, page)) return tail;
    tail.page = page;
    tail.count = p.c.counts_in[page];
    return tail;
  };
  // A thread's first child's: a chain of four loads, beside those of the marks.
  const int own = begin + int(threadIdx.x);
  const Tail of_own = own < end ? tail_of(own) : Tail{-1, -1, 0, 0};
  const int free_here = mark_pages<false>(p, sm, rank, p.c.counts_in, p.c.counts_in != p.c.counts_out ? p.c.counts_out : nullptr);
  cluster_wait();  // (all blocks run, and have written the above)
  tell(sm, 0, rank, free_here);
  for (int child = own; child < end; child += kThreads) {
    const int parent = child == own ? of_own.parent : p.parents[child];
    if (unsigned(parent) < unsigned(requests)) {
      atomicMin(p.first + parent, child);
      atomicAdd(p.heirs + parent, 1);
    }
  }
  meet();
  // Who wants a page: where the last page is partly filled, all but the first to continue a request, and that one too if others have named the page. (Told now: the
  // counts change below.)
  int wishes = 0;
  for (int child = own; child < end; child += kThreads) {
    const Tail tail = child == own ? of_own : tail_of(child);
    const bool wants = tail.page >= 0 && (__ldcg(p.first + tail.parent) != child || tail.count != 1);
    p.ranks[child] = wants ? -1 : kShared;
    wishes += wants;
  }
  wishes = block_sum(sm, wishes);
  tell(sm, 1, rank, wishes);
  const int free = in_all(sm, 0);
  list_marked(p, sm, rank, in_front(sm, 0, rank), children, [](uint32_t marks, int) { return marks; }, [&](int at, int page) { p.numbers[at] = page; });
  meet();  // (the last: nobody is told anything behind it)
  if (rank == 0 && threadIdx.x == 0) *p.copy_count = min(in_all(sm, 1), free);
  int rank_of_tile = in_front(sm, 1, rank);
  for (int tile = begin; tile < end; tile += kThreads) {
    const int child = tile + int(threadIdx.x);
    const bool wants = child < end && p.ranks[child] != kShared;
    int total;
    const int place = rank_of_tile + block_rank(sm, wants, &total);
    rank_of_tile += total;
    if (wants && place < free) {
      const int page = __ldcg(p.numbers + place);
      const Tail tail = child == own ? of_own : tail_of(child);
      p.ranks[child] = page;
      p.c.counts_out[page] = 1;
      p.copies[place] = make_int4(tail.page, page, tail.rows, 0);
    } else if (wants) {
      report(p.c.status, SPARSE_MLA_STATUS_NO_PAGE, child, extent_of(p, p.parents[child], p.c.lengths[p.parents[child]], false).entries - 1);
    }
  }
  if constexpr (kCopies) write_and_copy_here(all, rank);
}

// ---- compact --------------------------------------------------------------------------------------------------------

template <bool kCopies>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 1) compact_kernel(const __grid_constant__ Copies all) {
  const Plan& p = all.plan;
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  const int rank = int(cluster_rank()), blocks = int(p.c.blocks);
  wait_for_predecessor();
  let_successor_start();
  cluster_arrive_relaxed();
  const int used_here = mark_pages<true>(p, sm, rank, p.c.counts_in, p.c.counts_in != p.c.counts_out ? p.c.counts_out : nullptr);
  cluster_wait();  // (all blocks run)
  tell(sm, 0, rank, used_here);
  meet();
  const int border = in_all(sm, 0), used_in_front = in_front(sm, 0, rank);  // pages in use; those of them in front of this block's
  // Lists by number: pages in use from the border on, the first of them at the number of those in front of the border (`stay`); free pages in front of it from 0 on.
  auto movers = [&](uint32_t marks, int page0) { return marks & ~below(page0, border); };
  auto holes = [&](uint32_t marks, int page0) { return ~marks & below(page0, border); };  // (border <= blocks)
  int staying = 0;
  const int lane = threadIdx.x & 31;
  for (int word = threadIdx.x >> 5; word < p.words; word += kWarps) {
    const uint32_t marks = sm.marks[word];
    const int first = (rank * p.words + word) * 32, page = first + lane;
    staying += __popc(marks & below(first, border));
    const bool used = marks >> lane & 1;
    if (page < blocks && (!used || page < border)) p.places[page] = used ? page : -1;
  }
  staying = block_sum(sm, lane == 0 ? staying : 0);
  tell(sm, 1, rank, staying);
  int* const lists = reinterpret_cast<int*>(p.copies);
  // (pages in front of this block's that are free and in front of the border: all of those in front of the border but the ones in use)
  const int page0 = min(rank * p.words * 32, border), used_below = page0 < border ? used_in_front : 0;
  list_marked(p, sm, rank, used_in_front + staying, INT_MAX, movers, [&](int at, int page) { p.numbers[at] = page; });
  list_marked(p, sm, rank, page0 - used_below, INT_MAX, holes, [&](int at, int page) { lists[4 * at + 1] = page; });
  meet();  // (the last: nobody is told anything behind it)
  const int stay = in_all(sm, 1), moves = border - stay;
  if (rank == 0 && threadIdx.x == 0) *p.copy_count = moves;
  for (int move = rank * kThreads + threadIdx.x; move < moves; move += kCluster * kThreads) {
    const int source = __ldcg(p.numbers + stay + move), target = __ldcg(lists + 4 * move + 1);
    lists[4 * move] = source;
    lists[4 * move + 2] = int(p.c.page_rows);
    p.places[source] = target;
    p.c.counts_out[target] = p.c.counts_in[source];
    p.c.counts_out[source] = 0;
  }
  if constexpr (kCopies) write_and_copy_here(all, rank);
}

// ---- launch ---------------------------------------------------------------------------------------------------------

bool fits(const pages_call& c) {
  return c.requests >= 0 && c.requests < INT_MAX && c.entries >= 0 && c.entries < INT_MAX && (c.entries == 0 || c.requests <= INT_MAX / c.entries) && c.blocks >= 0 &&
         c.blocks <= PAGES_MOST_BLOCKS && c.page_rows >= 1 && c.page_rows <= INT_MAX;
}

// Where things lie in the workspace.
struct Layout {
  size_t bytes = 16;  // the number of copies
  size_t take(int64_t size) {
    const size_t at = bytes;
    bytes += (size_t(size) + 15) / 16 * 16;
    return at;
  }
};

int words_of(const pages_call& c) { return int((c.blocks + 32 * kCluster - 1) / (32 * kCluster)); }
// Up to so many units of a copy (in the worst case), and rows of a fork's tables, the planning blocks work through by themselves, one after the other by 32 groups of threads, which spares the host a launch. By them /
// by a second kernel, called eagerly, us (in brackets replayed from a graph, where a launch costs less than their copies): rows of one beam, none to copy 9.1 / 10.2 (9.2 / 9.3); 16 rows of four
// beams, 48 units 11.9 / 10.8 (11.9 / 9.4); compaction of a cache of 70 pages, 105 units 9.3 / 10.3 (9.2 / 6.8), of 100 pages, 150 units 10.6 / 10.4 (10.5 / 6.8); 192 units, fork 14.4 / 11.1, 420,
// compaction 15.0 / 11.0, 1000 of 1152 bytes 23.9 / 10.5. Rows alone, 32 of 32 requests 9.4 / 10.4, 64 of 64 11.6 / 10.7, 256 of 256 25.7 / 11.9, 2000 of 2000 141 / 18.6; 48 units, 16 of 512 24.2 / 10.8.
constexpr int64_t kFewItems = 160;

template <class Arguments>
int launch_plan(void (*kernel)(const Arguments), const Arguments& arguments, const Plan& p, cudaStream_t stream) {
  const size_t shared = sizeof(Shared) + size_t(p.words) * sizeof(uint32_t);
  if (shared + sizeof(uint16_t) * kWarps * kStaged > 48 * 1024)  // (a per-device setting; always the same value)
    if (const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Shared) + PAGES_MOST_BLOCKS / 8 / kCluster))) return int(error);
  return int(launch_overlapped(kernel, kCluster, kThreads, shared, stream, arguments));
}

int fill_tensors(Copies* copies, const pages_call& c, const pages_tensor* tensors, int64_t count) {
  if (count < 0 || count > PAGES_MOST_TENSORS || (count > 0 && tensors == nullptr)) return -1;
  int64_t units = 0;
  for (int64_t t = 0; t < count; ++t) {
    const pages_tensor& own = tensors[t];
    if (own.page_bytes < 0 || own.rows < 1 || own.rows > c.page_rows || c.page_rows % own.rows != 0 || own.page_bytes % own.rows != 0) return -1;
    copies->tensor[t] = {static_cast<char*>(own.memory), own.page_bytes, int32_t(own.rows), int32_t(units)};
    units += std::max<int64_t>((own.page_bytes + kUnitBytes - 1) / kUnitBytes, 1);
    if (units > INT_MAX) return -1;
  }
  copies->tensors = int32_t(count);
  copies->units = int32_t(units);
  copies->page_rows = c.page_rows;
  return 0;
}

int launch_copies(const Copies& copies, int64_t most, cudaStream_t stream) {
  const int64_t items = std::max({most * copies.units, copies.forks ? std::max<int64_t>(copies.plan.children, copies.plan.c.requests) : 0, (copies.entries + kCopyThreads - 1) / kCopyThreads});
  if (items == 0) return 0;
  const int grid = int(std::min<int64_t>(items, int64_t(latent::multiprocessors()) * kCopyBlocks));
  return int(launch_overlapped(copy_kernel, grid, kCopyThreads, 0, stream, copies));
}

bool usable(const pages_call& c) { return c.workspace != nullptr && latent::aligned(c.workspace) && c.status != nullptr; }

}  // namespace
}  // namespace pages

extern "C" {

int workspace_size_pages_resize(uint64_t* bytes, const pages_call* call) {
  using namespace pages;
  if (bytes == nullptr || call == nullptr || !fits(*call)) return -1;
  Layout layout;
  layout.take(4 * call->blocks);
  for (int i = 0; i < 3; ++i) layout.take(4 * call->requests);
  layout.take(4 * kCluster * int64_t(words_of(*call)));
  *bytes = layout.bytes;
  return 0;
}

int launch_pages_resize(void* stream, const pages_call* call) {
  using namespace pages;
  if (call == nullptr || !fits(*call)) return -1;
  if (call->requests == 0 && (call->blocks == 0 || call->counts_in == call->counts_out)) return 0;  // (requests of a table without entries may have lengths to report)
  if (!usable(*call)) return -1;
  char* workspace = static_cast<char*>(call->workspace);
  Plan p = {};
  Layout layout;
  p.c = *call;
  p.numbers = reinterpret_cast<int32_t*>(workspace + layout.take(4 * call->blocks));
  p.first = reinterpret_cast<int32_t*>(workspace + layout.take(4 * call->requests));
  p.heirs = reinterpret_cast<int32_t*>(workspace + layout.take(4 * call->requests));
  p.ranks = reinterpret_cast<int32_t*>(workspace + layout.take(4 * call->requests));
  p.marks = reinterpret_cast<uint32_t*>(workspace + layout.take(4 * kCluster * int64_t(words_of(*call))));
  p.free = reinterpret_cast<int32_t*>(workspace);
  const int64_t entries = call->requests * call->entries;
  p.words = words_of(*call);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (entries <= kSmallTable && call->entries <= kShortRow) return launch_plan(resize_kernel, p, p, s);
  if (call->counts_in != call->counts_out && call->blocks > 0) {
    const int64_t grid = std::min<int64_t>((call->blocks + kRowThreads * 8 - 1) / (kRowThreads * 8), latent::multiprocessors() * 4);
    if (const cudaError_t error = launch_overlapped(copy_counts_kernel, int(grid), kRowThreads, 0, s, p)) return int(error);
  }
  if (const cudaError_t error = launch_overlapped(release_kernel, int(call->requests), kRowThreads, 0, s, p)) return int(error);
  if (call->blocks > kManyPages) {
    const int grid = (kCluster * p.words + kRowThreads / 32 * kWordsPerWarp - 1) / (kRowThreads / 32 * kWordsPerWarp);
    if (const cudaError_t error = launch_overlapped(mark_kernel, grid, kRowThreads, 0, s, p)) return int(error);
  } else {
    p.marks = nullptr;
  }
  if (const int status = launch_plan(rank_kernel, p, p, s)) return status;
  return int(launch_overlapped(give_kernel, int(call->requests), kRowThreads, 0, s, p));
}

int workspace_size_pages_fork(uint64_t* bytes, const pages_fork_call* call) {
  using namespace pages;
  if (bytes == nullptr || call == nullptr || !fits(call->pages) || call->children < 0 || call->children >= INT_MAX) return -1;
  Layout layout;
  layout.take(4 * call->children);
  layout.take(4 * call->pages.requests);
  layout.take(4 * call->pages.requests);
  layout.take(16 * call->children);
  layout.take(4 * call->children);
  *bytes = layout.bytes;
  return 0;
}

int launch_pages_fork(void* stream, const pages_fork_call* call) {
  using namespace pages;
  if (call == nullptr || !fits(call->pages) || call->children < 0 || call->children >= INT_MAX) return -1;
  const pages_call& c = call->pages;
  if (c.entries > 0 && call->children > INT_MAX / c.entries) return -1;
  Copies copies = {};
  if (const int status = fill_tensors(&copies, c, call->tensors, call->tensor_count)) return status;
  if (c.requests == 0 && (call->children == 0 || c.entries == 0) && (c.blocks == 0 || c.counts_in == c.counts_out)) return 0;
  if (!usable(c)) return -1;
  char* workspace = static_cast<char*>(c.workspace);
  Plan p = {};
  Layout layout;
  p.c = c;
  p.parents = call->parents;
  p.children = int32_t(call->children);
  p.numbers = reinterpret_cast<int32_t*>(workspace + layout.take(4 * call->children));
  p.first = reinterpret_cast<int32_t*>(workspace + layout.take(4 * c.requests));
  p.heirs = reinterpret_cast<int32_t*>(workspace + layout.take(4 * c.requests));
  p.copies = reinterpret_cast<int4*>(workspace + layout.take(16 * call->children));
  p.ranks = reinterpret_cast<int32_t*>(workspace + layout.take(4 * call->children));
  p.copy_count = reinterpret_cast<int32_t*>(workspace);
  const int64_t entries = std::max(c.requests, call->children) * std::max<int64_t>(c.entries, 1);
  const bool few = call->children * copies.units + call->children + c.requests <= kFewItems && entries <= kSmallTable;
  p.words = words_of(c);
  copies.plan = p;
  copies.forks = true;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (few) return launch_plan(fork_kernel<true>, copies, p, s);
  if (const int status = launch_plan(fork_kernel<false>, copies, p, s)) return status;
  return launch_copies(copies, call->children, s);
}

int workspace_size_pages_compact(uint64_t* bytes, const pages_compact_call* call) {
  using namespace pages;
  if (bytes == nullptr || call == nullptr || !fits(call->pages)) return -1;
  Layout layout;
  layout.take(16 * (call->pages.blocks / 2 + 1));
  layout.take(4 * call->pages.blocks);
  *bytes = layout.bytes;
  return 0;
}

int launch_pages_compact(void* stream, const pages_compact_call* call) {
  using namespace pages;
  if (call == nullptr || !fits(call->pages)) return -1;
  const pages_call& c = call->pages;
  Copies copies = {};
  if (const int status = fill_tensors(&copies, c, call->tensors, call->tensor_count)) return status;
  const bool table = c.requests > 0 && c.entries > 0;
  if (c.blocks == 0 && (!table || c.table_in == c.table_out)) return 0;
  if (!usable(c)) return -1;
  char* workspace = static_cast<char*>(c.workspace);
  Plan p = {};
  Layout layout;
  p.c = c;
  p.places = call->places;
  p.copies = reinterpret_cast<int4*>(workspace + layout.take(16 * (c.blocks / 2 + 1)));  // (no more moves than free pages, or than pages in use)
  p.numbers = reinterpret_cast<int32_t*>(workspace + layout.take(4 * c.blocks));
  p.copy_count = reinterpret_cast<int32_t*>(workspace);
  copies.entries = table ? c.requests * c.entries : 0;
  const bool few = c.blocks / 2 * copies.units <= kFewItems && copies.entries <= kSmallTable;
  p.words = words_of(c);
  copies.plan = p;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (few) return launch_plan(compact_kernel<true>, copies, p, s);
  if (const int status = launch_plan(compact_kernel<false>, copies, p, s)) return status;
  return launch_copies(copies, c.blocks / 2, s);
}

}  // extern "C"
