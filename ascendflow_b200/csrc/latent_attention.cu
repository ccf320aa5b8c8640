// Attention over the paged latent cache in absorbed form: one row per token is key and value of all heads.
//
// out = softmax(scale Q X^T) X[:, :512] per request, Q the queries of all heads (row j * H + h), X the cached rows, row j * H + h seeing
// the first L - n + j + 1 of them. Rows of a request are dealt in tiles of 64, whatever the number of heads, and cached rows in
// chunks of 64 (pages are multiples). A block works on a stretch of the call's (tile, chunk) pairs, tile by tile: all blocks get
// stretches of the same cost (`plan_block`), so a tile may be shared by several blocks; their unnormalised sums then go to the
// workspace in FP32 and `combine_kernel` adds them up, in the order of the chunks.
//
//   warps 0-3   softmax: scores out of tensor memory, running reference and sum in FP32, P (16 bits) to shared memory, rescaling of
//               the accumulator, output.
//   warp 4      one thread issues S = Q X^T: Q from tensor memory, X K-major from the chunk's tile. 64 rows fill half of the 128 lanes
//               that the tensor core wants, so the features of a row are split between two lanes: lanes 0-15 of every subpartition
//               hold the even pairs of features of 16 rows, lanes 16-31 the odd pairs. Either is a 2:4 sparse row: W / 32 sparse
//               instructions M = 128, N = 64, K = 32 give every lane the partial scores of its pairs.
//   warp 5      one thread issues O += P X: weight-stationary M = 64, N = 256, X MN-major from the same tile.
//   warp 6      brings chunks by tensor copies (boxes of 64 features x 64 rows) into a ring of three tiles.
//   warp 7      works out the block's pieces (a tile and a stretch of its chunks) ahead of everybody.
//   warps 8-15  Q of the next piece from global to tensor memory, through registers.
//
// Tensor memory: columns 0-255 O (lane l: row l % 64, accumulators of features 128 (l / 64) .. + 127 and 256 more), 256-383 Q's first 512
// features, 384-447 scores, 448-463 the sparse products' metadata, 464-479 Q's other 64 features.
//
// What bounds it: memory where a request brings one token (64 requests of 64 heads at 32K: 2.42 GB in 380 us in a few calls after a pause, 6.4 TB/s;
// in a long loop 410-465 us at 1.0 GHz, since reading random data at that rate takes the board's 1000 W by itself: a plain reduction of as
// many bytes takes 393 us there), products where it brings several (32 requests of six tokens at 16K: 455-490 us, 0.9 PFLOP/s, 1.0 where all
// requests share their pages). A chunk takes 2.0 k cycles, 1.43 k of them the two products' own; shared memory's ports are busy for
// two thirds of it. Two tiles of weights (room for them by a ring of its own for the last 64 features), weights without looking for the
// maximum, and fewer barriers per chunk were each built and slower by 2 to 12 per cent in loops.
// A call of few chunks is a chain of 16 us: plan 2.5, pieces and page 0.8, copy 2.2, chunks 0.8 each, last products 0.5, sums to memory 1.8 (128 KiB
// per block), the next kernel's start 2.3, their sum 3.3.
//
// Rows of a chunk behind the request's length are cleared in the tile's value part (a zero weight times infinity is a
// NaN) and their scores replaced; so are whole chunks whose page is not in the cache, which are reported.
#include "latent_common.cuh"
#include "latent_parts.cuh"
#include "latent_ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace latent {
namespace absorbed {

using namespace sm100;

constexpr int kRows = 64, kChunk = 64;
constexpr int kSoftmaxWarps = 4, kScoreWarp = 4, kValueWarp = 5, kCopyWarp = 6, kPlanWarp = 7, kQueryWarp0 = 8, kQueryWarps = 8;
constexpr int kThreads = 32 * (kQueryWarp0 + kQueryWarps);
constexpr int kBoxBytes = kChunk * 128;  // 64 features of a chunk
constexpr int kStages = 3;
constexpr int kPieces = 4;               // pieces announced ahead
constexpr int kSpoilt = 128;             // see Shared::marked

constexpr uint32_t kColumnsQ = 256, kColumnsScores = 384, kColumnsPlaces = 448, kColumnsQRest = 464;
constexpr uint32_t kHighLanes = 16u << 16;

// What a block does next: rows of one request's tile and a stretch of chunks.
struct Piece {
  int64_t row;      // first row of q and out
  int rows;         // 1 .. 64
  int request;
  int token;        // the tile's first row's token within the request
  int head;         // ... and head
  int base;         // keys that the request's first token sees: L - n + 1
  int length;       // keys of the request that may be read
  int first, last;  // chunks [first, last); first < 0: no more pieces
  int slot;         // of the workspace, or -1: the piece is all of its tile
};
static_assert(sizeof(Piece) <= 64, "the piece ring holds 64-byte entries");

template <int kWidth>
struct Layout {
  static constexpr int kBoxes = kWidth / 64;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kSmemP = kStages * kTileBytes;            // 64 rows x 64 weights; the output on its way out
  static constexpr int kSmemPieces = kSmemP + kRows * 128;
  static constexpr int kSmemBars = kSmemPieces + kPieces * 64;
  static constexpr int kSmemAlpha = kSmemBars + 320;             // float[2][64]
  static constexpr int kSmemInverse = kSmemAlpha + 2 * kRows * 4;  // float[64]
  static constexpr int kSmemMisc = kSmemInverse + kRows * 4;
  static constexpr int kSmemScales = kSmemMisc + 64;             // bytes[3][64], of rows in 8 bits
  static constexpr int kSmemBytes = kSmemScales + kStages * kChunk + 1024;  // the tiles are aligned to 1024 bytes
};
static_assert(Layout<576>::kSmemBytes <= 232448, "one block per SM");

enum Bar {
  kFull0 = 0, kFree0 = kFull0 + kStages, kPieceReady0 = kFree0 + kStages, kPieceDone0 = kPieceReady0 + kPieces, kQFull = kPieceDone0 + kPieces,
  kQFree, kPlaces, kScoresFull, kScoresFree, kWeightsFull, kWeightsFree, kMended, kGivenUp0, kGivenUp1, kLanded0, kFreeHalf0 = kLanded0 + 2 * kStages,
  kBarCount = kFreeHalf0 + kStages
};
static_assert(kBarCount <= 40, "the barrier area");

// Workspace: per block a record, statistics and sums of two slots (2 i: a tile that begins in an earlier block; 2 i + 1: one that begins here and
// ends in a later one).
struct Record {
  int64_t row;
  int rows, head;
  int last;       // block that has the tile's end; -1: no tile begins here that ends elsewhere
  int pad[3];
};
constexpr int kSlotFloats = kRows * LATENT_VALUES;
// Sums of eight features of 32 rows lie next to each other, as warps write them: 32 bytes to a row, 1 KiB to an instruction (in rows, a write
// touched 32 lines, and 128 KiB took 3.6 us instead of 1.8). First feature of eight.
__device__ __forceinline__ int sums_place(int row, int feature) {
  return ((((feature >> 7 & 1) * 2 + (row >> 5)) * 32 + (feature >> 8) * 16 + (feature & 127) / 8) * 32 + (row & 31)) * 8;
}
inline size_t statistics_offset(int blocks) { return size_t(blocks) * sizeof(Record); }
inline size_t sums_offset(int blocks) { return (statistics_offset(blocks) + size_t(blocks) * 2 * kRows * sizeof(float2) + 511) / 512 * 512; }
inline size_t workspace_bytes(int blocks) { return sums_offset(blocks) + size_t(blocks) * 2 * kSlotFloats * sizeof(float); }

// x / divisor for x from 0 to 2^31 - 1 (exact: 2^shift / divisor is rounded up by less than 2^-31 of it). A division by a number that is not known takes
// 130 cycles, in a chain that the whole call waits for.
struct Divisor {
  uint32_t factor;
  int32_t shift;
};
inline Divisor divisor_of(int divisor) {
  int bits = 0;
  while ((int64_t(1) << bits) < divisor) ++bits;
  return {uint32_t((uint64_t(1) << (31 + bits)) / uint32_t(divisor) + 1), 31 + bits};
}
__device__ __forceinline__ int over(int x, const Divisor& by) { return int(uint64_t(uint32_t(x)) * by.factor >> by.shift); }

struct Params {
  CUtensorMap cache;
  CUtensorMap rest;  // rows in 8 bits: their last 64 features
  const char* q;
  const int32_t *table, *cu, *lengths;
  const float* sinks;
  char* out;
  float* lse;
  Record* records;
  float2* statistics;
  float* sums;
  int32_t* status;
  int32_t batches, tokens, heads, pages, blocks, page_rows;
  Divisor by_heads, by_page;  // a page's chunks
  int32_t tile_tokens;        // that a tile's rows belong to, at most
  float scale_log2;
  const char* held;           // rows in 8 bits, and their scales
  const uint8_t* scales;
  int32_t block_shift;        // 2^this rows share a scale
};

struct Shared {
  uint32_t base;
  unsigned char* ptr;
  int bars, pieces, misc;
  __device__ __forceinline__ uint32_t bar(int which) const { return base + bars + which * 8; }
  __device__ __forceinline__ Piece* piece(uint32_t index) const { return reinterpret_cast<Piece*>(ptr + pieces + (index % kPieces) * 64); }
  __device__ __forceinline__ uint32_t* tmem_slot() const { return reinterpret_cast<uint32_t*>(ptr + misc); }
  __device__ __forceinline__ volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(ptr + misc + 4); }
  __device__ __forceinline__ volatile int* live(uint32_t stage) const { return reinterpret_cast<volatile int*>(ptr + misc + 8 + stage * 4); }
  // Rows in 8 bits: the same, less kSpoilt where a scale among them is NaN (so that what looks out for a chunk's end finds it); which, of keys 32 half .. + 31.
  __device__ __forceinline__ volatile int* marked(uint32_t stage) const { return reinterpret_cast<volatile int*>(ptr + misc + 20 + stage * 4); }
  __device__ __forceinline__ volatile uint32_t* spoilt(uint32_t stage, int half) const { return reinterpret_cast<volatile uint32_t*>(ptr + misc + 32 + (stage * 2 + half) * 4); }
  __device__ __forceinline__ int64_t* scan() const { return reinterpret_cast<int64_t*>(ptr); }  // (before the first tile lands)
};

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit = 1ll << 31) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit));
}

// ---- the plan -----------------------------------------------------------------------------------------------------

// A request's tiles and what they cost, in cached rows: kFixed for a tile, and the keys that its rows see, from `near` on up to `far`.
constexpr int kFixed = 128;

struct Request {
  int begin, count;  // tokens
  int length;        // keys
  int rows, tiles;
  int seen;          // keys that may be read, and one behind the table where the length does not fit
  int near, far, fixed;
  // Cost of the first `t` tiles: any function will do that everybody evaluates alike and that grows.
  __device__ __forceinline__ int64_t cost(int t) const {
    int64_t sum = int64_t(t) * (fixed + near);
    if (far != near) sum += int64_t(far - near) * (int64_t(t) * (t - 1) / 2) / (tiles - 1);  // (below 2^31 x 2^31; more than one tile)
    return sum;
  }
  // Blocks that a tile gets if each takes 1 / `density` rows or a little less (rounded somehow: only everybody has to get the same).
  __device__ __forceinline__ int blocks(float density) const { return max(1, int(ceilf(float(far) * density))); }
  // From here on a tile costs the blocks that it gets.
  __device__ __forceinline__ void dealt(float density) {
    near = far = blocks(density);
    fixed = 0;
  }
};

__device__ __forceinline__ Request request_at(const Params& p, int b, float density = 0.f) {
  Request r;
  r.begin = min(max(p.cu[b], 0), p.tokens);
  r.count = max(min(max(p.cu[b + 1], 0), p.tokens) - r.begin, 0);
  r.length = max(p.lengths[b], 0);
  r.rows = r.count * p.heads;
  r.tiles = (r.rows + kRows - 1) / kRows;
  // (one key behind the table is enough to report a length that does not fit)
  r.seen = r.far = int(min(int64_t(r.length), int64_t(p.pages) * p.page_rows + 1));
  r.near = int(min(int64_t(r.far), max(int64_t(r.length) - r.count, int64_t(0)) + p.tile_tokens));
  // Nearly alike (as where tokens are decoded), or too many for the product in `cost`: taken to be alike, which spares a division.
  if (r.far - r.near <= kChunk) r.near = r.far;
  else if (r.tiles > 65536) r.near = r.far = (r.near >> 1) + (r.far >> 1);
  r.fixed = kFixed;
  if (density > 0.f) r.dealt(density);
  return r;
}

// Chunks that tile t's rows see.
__device__ __forceinline__ int chunks_of(const Params& p, const Request& r, int t) {
  const int last_token = over(min((t + 1) * kRows, r.rows) - 1, p.by_heads);
  const int64_t seen = int64_t(r.length) - r.count + last_token + 1;
  return int((min(max(seen, int64_t(0)), int64_t(r.seen)) + kChunk - 1) / kChunk);
}

// Stretch [at(i), at(i + 1)) of the total cost is block i's.
struct Borders {
  int64_t total, each;
  uint32_t rest, blocks;  // that get a stretch (at most 255)
  bool whole;             // stretches end between tiles
  float density;          // > 0: every tile has blocks of its own, so many per row; costs are numbers of blocks
  float inverse;          // 1 / blocks
  __device__ __forceinline__ int64_t at(uint32_t i) const { return each * i + int(fmaf(float(rest * i), inverse, 0.001f)); }  // (the quotient rounded down: both are at most 255)
};
// Quotients of numbers that are not negative (a 64-bit division takes several times as long as one of 32 bits).
__device__ __forceinline__ int64_t quotient(int64_t value, int64_t divisor) {
  if ((uint64_t(value) | uint64_t(divisor)) >> 32 == 0) return uint32_t(value) / uint32_t(divisor);
  return value / divisor;
}
// value * factor / divisor, rounded down or nearly so, for value <= divisor: everybody who asks gets the same, and more for a larger value.
__device__ __forceinline__ int share_of(int64_t value, int factor, int64_t divisor) {
  return min(int(fmaf(float(value), float(factor) / float(divisor), 0.001f)), factor);
}
// What sharing tiles costs a call, in cached rows: the parts' way through memory and `combine_kernel`, the more of both the more tiles there are to share.
// Where giving every tile to one block makes no block's stretch longer than that, none is shared: the borders move to the nearest tile's. (64 heads, one
// token, whole / shared: 512 keys 16.0 / 13.3 us, 16 requests of 512 16.9 / 15.9, 32 of 768 20.4 / 19.6, 64 of 1024 27.5 / 32.9, of 1500 41.3 / 42.5,
// of 2048 48.9 / 48.6.)
constexpr int kSharing = 4 * kChunk, kSharingMany = 28 * kChunk;
// A block that ends one tile and begins another writes sums twice, and all wait for it. Where every tile can have blocks of its own without making the
// stretches longer than by this (for 64 rows), it has: 64 heads, one token, 3, 8, 16, 32 requests of 8192 keys 21.7, 29.5, 45.8, 74.4 us with borders anywhere,
// 19.8, 27.4, 44.5, 71.8 so; 4, 16, 64 requests of 1024 to 8192 keys 22.2, 32.2, 89.3 and 19.5, 29.7, 85.3.
constexpr int kTwoTiles = 10 * kChunk;
// A block with fewer chunks than these loses more with its start and with its part of the sums than it takes off the others (64 heads, one
// token; 1, 2, 3 chunks: 512 keys 13.8, 13.4, 13.8 us, 2048 14.1, 14.4, 14.7, 8192 18.1, 16.1, 16.3, four requests of 8192 20.6 each).
constexpr int kLeastChunks = 2;

// Where a stretch begins: a request's tile and the cost in front of that.
struct Place {
  int request, tile;
  int64_t start;
};

// Sum over the threads that plan, for all of them: a block's, or a warp's.
template <int kWarps>
__device__ __forceinline__ int64_t plan_sum(int64_t value, int64_t* scratch) {
  if constexpr (kWarps == 1)  // up to 32 requests: below 2^56
    return (int64_t(__reduce_add_sync(0xffffffffu, uint32_t(value >> 27))) << 27) + __reduce_add_sync(0xffffffffu, uint32_t(value) & ((1u << 27) - 1));
  else {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) value += __shfl_xor_sync(0xffffffffu, value, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = value;
    __syncthreads();
    int64_t sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += scratch[w];
    return sum;
  }
}

// The same for numbers whose sum fits.
template <int kWarps>
__device__ __forceinline__ int plan_count(int value, int64_t* scratch) {
  value = __reduce_add_sync(0xffffffffu, value);
  if constexpr (kWarps == 1) return value;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = value;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += int(scratch[w]);
  return sum;
}

// The stretches, and where this block's begins; by all threads of the block, or, for up to 32 requests, by one warp (which saves the others' barriers:
// 1.1 of 21.5 us of a call of one token).
//
// The order of the tiles: the first tile of every request, then the second ones, and so on. Where requests have as many tiles each, and
// the blocks are a multiple of that, the blocks that work on a request's tiles go through its chunks side by side: a chunk comes from
// memory once and from L2 for the others. (Tile after tile they would be chunks apart: 32 requests of 6 tiles and 256 chunks then
// read 3.6 GB instead of 0.6.) Up to a sixteenth of the blocks is given up for that.
template <int kWarps>
__device__ __forceinline__ Borders plan_block(const Params& p, int64_t* scratch, Place* place) {
  constexpr int kRound = 32 * kWarps;  // requests at a time
  const int warp = kWarps == 1 ? 0 : int(threadIdx.x >> 5), lane = threadIdx.x & 31, thread = warp * 32 + lane;
  const int rounds = (p.batches + kRound - 1) / kRound;
  Request none = {};
  Borders borders = {0, 0, 0, 0, false, 0.f, 0.f};
  Request own = thread < p.batches ? request_at(p, thread) : none;
  auto of_round = [&](int round) {
    const int b = round * kRound + thread;
    return round == 0 ? own : b < p.batches ? request_at(p, b) : none;
  };
  int64_t cost = 0;
  int most_tiles = 0, least_tiles = INT32_MAX, most_cost = 0, least_cost = INT32_MAX;
  for (int round = 0; round < rounds; ++round) {
    const Request r = of_round(round);
    cost += r.cost(r.tiles);
    most_tiles = max(most_tiles, r.tiles);
    if (r.tiles > 0) {
      least_tiles = min(least_tiles, r.tiles);
      most_cost = max(most_cost, r.far);
      least_cost = min(least_cost, r.near);
    }
  }
  most_tiles = __reduce_max_sync(0xffffffffu, most_tiles);
  least_tiles = __reduce_min_sync(0xffffffffu, least_tiles);
  most_cost = __reduce_max_sync(0xffffffffu, most_cost);
  least_cost = __reduce_min_sync(0xffffffffu, least_cost);
  if (kWarps > 1 && lane == 0) {
    scratch[kWarps + warp] = int64_t(most_tiles) << 32 | uint32_t(least_tiles);
    scratch[2 * kWarps + warp] = int64_t(most_cost) << 32 | uint32_t(least_cost);
  }
  borders.total = plan_sum<kWarps>(cost, scratch);
#pragma unroll
  for (int w = 0; w < (kWarps > 1 ? kWarps : 0); ++w) {
    most_tiles = max(most_tiles, int(scratch[kWarps + w] >> 32));
    least_tiles = min(least_tiles, int(uint32_t(scratch[kWarps + w])));
    most_cost = max(most_cost, int(scratch[2 * kWarps + w] >> 32));
    least_cost = min(least_cost, int(uint32_t(scratch[2 * kWarps + w])));
  }
  if (borders.total == 0) return borders;
  const int grid = int(gridDim.x), most = most_cost + kFixed;
  int blocks = int(min(max(borders.total / (kLeastChunks * kChunk), int64_t(1)), int64_t(grid)));
  const bool alike = most_cost == least_cost;
  const float total = float(borders.total), part = 1.f / float(grid), mean = total / float(blocks), tiles = total / float(most);  // (tiles: where all cost the same)
  // The longest stretch if no tile is shared: whole rounds where all cost the same, otherwise half a tile more than the mean, and a tile at least.
  const float longest = alike ? ceilf(tiles * part - 0.003f) * float(most) : fmaxf(float(most), total * part + 0.5f * float(most));
  borders.whole = longest <= mean + float(kSharing) + float(kSharingMany) * fminf(tiles * part, 1.f);
  static_assert(kWarps == 1 || kRound > 255, "a thread for each of as many requests as blocks");
  if (!borders.whole && tiles < float(grid) + 0.5f && p.batches <= grid && mean < float(1 << 30)) {  // blocks of their own for every tile?
    const float rows = fminf(float(kRows), float(p.tokens * p.heads) / float(p.batches));
    const int more = int(float(kTwoTiles / kRows) * rows);  // (what a second tile costs is its rows' sums)
    if (alike) {
      const int each = min(int(float(grid) / tiles + 0.001f), int(uint32_t(most_cost + kLeastChunks * kChunk - 1) / (kLeastChunks * kChunk)));
      if ((mean + float(more)) * float(each) * tiles >= total) blocks = each * int(tiles + 0.5f);
    } else {
      // The shortest stretch that will do, nearly.
      int needed = 0, stretch = 0;
#pragma unroll 1
      for (int candidate = int(mean), step = more;;) {
        const float tried = 1.f / float(candidate);
        // (a request's tiles have to cost the same; each thread has a request at most)
        const int wanted = own.near == own.far && own.tiles <= grid ? own.tiles * min(own.blocks(tried), grid + 1) : grid + 1;
        const int sum = plan_count<kWarps>(own.tiles == 0 ? 0 : wanted, scratch);
        if (sum <= grid) {
          stretch = candidate;
          borders.density = tried;
          needed = sum;
        }
        if (candidate == int(mean)) {
          if (stretch > 0 || more == 0) break;
          candidate += more;
        } else {
          step >>= 1;
          if (stretch == 0 || step < kChunk / 3) break;
          candidate = stretch - step;
        }
      }
      if (stretch > 0) {
        borders.total = blocks = needed;
        if (thread < p.batches) own.dealt(borders.density);
      }
    }
  }
  if (borders.density == 0.f && most_tiles == least_tiles && most_tiles > 1 && uint32_t(blocks) % uint32_t(most_tiles) <= uint32_t(blocks) / 16) blocks -= uint32_t(blocks) % uint32_t(most_tiles);
  if (int(blockIdx.x) >= blocks) return borders;
  borders.blocks = uint32_t(blocks);
  borders.inverse = 1.f / float(blocks);
  borders.each = borders.density > 0.f ? 1 : quotient(borders.total, blocks);
  borders.rest = uint32_t(borders.total - borders.each * blocks);
  const int64_t mine = borders.at(blockIdx.x);
  // The tile: the last whose predecessors cost no more.
  int tile = 0;
  int64_t passed = 0;
  for (int high = most_tiles; high - tile > 1;) {
    const int middle = (tile + high) >> 1;
    int64_t before = 0;
    for (int round = 0; round < rounds; ++round) {
      const Request r = of_round(round);
      before += r.cost(min(middle, r.tiles));
    }
    before = plan_sum<kWarps>(before, scratch);
    if (before <= mine) {
      tile = middle;
      passed = before;
    } else {
      high = middle;
    }
  }
  // The request.
  for (int round = 0; round < rounds; ++round) {
    const Request r = of_round(round);
    const int64_t value = r.tiles > tile ? r.cost(tile + 1) - r.cost(tile) : 0;
    int64_t inclusive = value;
    if (borders.total <= INT32_MAX) {
      int few = int(value);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, few, d);
        if (lane >= d) few += other;
      }
      inclusive = few;
    } else {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t other = __shfl_up_sync(0xffffffffu, inclusive, d);
        if (lane >= d) inclusive += other;
      }
    }
    int64_t sum = 0, in_front = 0;
    if constexpr (kWarps > 1) {
      __syncthreads();
      if (lane == 31) scratch[warp] = inclusive;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) in_front = sum;
        sum += scratch[w];
      }
    }
    const int64_t start = passed + in_front + inclusive - value;
    const bool mine_begins = value > 0 && start <= mine && mine < start + value;
    if constexpr (kWarps == 1) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, mine_begins)) - 1;
      *place = {owner, tile, __shfl_sync(0xffffffffu, start, owner & 31)};
      return borders;  // (one round)
    }
    if (mine_begins) {
      scratch[3 * kWarps] = round * kRound + thread;
      scratch[3 * kWarps + 1] = start;
    }
    passed += sum;
  }
  if constexpr (kWarps > 1) {
    __syncthreads();
    *place = {int(scratch[3 * kWarps]), tile, scratch[3 * kWarps + 1]};
  }
  return borders;
}

// The pieces of this block, announced one after the other (by one warp; all lanes work out the same).
__device__ void plan_role(const Params& p, const Shared& sm, const Borders& borders, const Place& place) {
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  Record record = {0, 0, 0, -1, {0, 0, 0}};
  bool continued = false;  // slot 2 i holds a part of the tile before
  uint32_t announced = 0;
  // A free entry of the ring; false when somebody has given up.
  auto claim = [&]() { return announced < kPieces || warp_wait(sm.bar(kPieceDone0 + announced % kPieces), (announced / kPieces - 1) & 1, abort_flag, kLongWait); };
  auto announce = [&](const Piece& piece) {
    if (lane == 0) {
      *sm.piece(announced) = piece;
      mbar_arrive(sm.bar(kPieceReady0 + announced % kPieces));
    }
    ++announced;
  };
  if (borders.blocks > 0) {
    const int64_t end = borders.at(blockIdx.x + 1);
    int64_t at = borders.at(blockIdx.x);
    int request = place.request, tile = place.tile;
    int64_t start = place.start;
    while (at < end) {
      const Request r = request_at(p, request, borders.density);
      const int64_t cost = r.cost(tile + 1) - r.cost(tile), past = start + cost;
      const int chunks = chunks_of(p, r, tile);
      Piece piece;
      if (borders.whole) {  // a border belongs to the tile's nearer end
        const bool begins = 2 * (at - start) < cost, ends = past <= end || 2 * (end - start) >= cost;
        piece.first = begins ? 0 : chunks;
        piece.last = begins && ends ? chunks : 0;
        if (begins && ends) at = start;
        else if (chunks == 0) at = start + 1;
      } else {
        piece.first = at == start ? 0 : share_of(at - start, chunks, cost);
        piece.last = past <= end ? chunks : share_of(end - start, chunks, cost);
      }
      if (piece.first < piece.last || (chunks == 0 && at == start)) {
        const int row = tile * kRows;
        piece.row = int64_t(r.begin) * p.heads + row;
        piece.rows = min(kRows, r.rows - row);
        piece.request = request;
        piece.token = over(row, p.by_heads);
        piece.head = row - piece.token * p.heads;
        piece.base = r.length - r.count + 1;
        piece.length = r.seen;
        const bool whole = piece.first == 0 && piece.last == chunks;
        piece.slot = whole ? -1 : 2 * int(blockIdx.x) + (piece.first == 0);
        if (!claim()) break;
        announce(piece);
        if (!whole && piece.first == 0) {
          record.row = piece.row;
          record.rows = piece.rows;
          record.head = piece.head;
          // The block that has the tile's end: the last that begins in front of it.
          int last = blockIdx.x;
          for (int high = int(borders.blocks); high - last > 1;) {
            const int middle = (last + high) >> 1;
            if (borders.at(middle) < past) last = middle; else high = middle;
          }
          record.last = last;
        } else if (!whole) {
          continued = true;
        }
      }
      at = min(past, end);
      if (at >= end) break;
      // The next request that has such a tile, or the first that has one more.
      start = past;
      unsigned hit = 0;
      for (int turn = 0; turn < 2 && hit == 0; ++turn) {
        for (int b = turn == 0 ? request + 1 : 0; hit == 0 && b < p.batches; b += 32) {
          hit = __ballot_sync(0xffffffffu, b + lane < p.batches && request_at(p, b + lane).tiles > tile);
          if (hit != 0) request = b + __ffs(hit) - 1;
        }
        if (hit == 0) ++tile;
      }
      if (hit == 0) break;  // (does not happen: there is cost left)
    }
  }
  if (lane == 0) p.records[blockIdx.x] = record;
  if (!continued)
    for (int row = lane; row < kRows; row += 32) p.statistics[size_t(2 * blockIdx.x) * kRows + row] = make_float2(-INFINITY, 0.f);
  if (!claim()) return;
  Piece none = {};
  none.first = -1;
  announce(none);
}

// Everybody's way through the pieces. `next` waits for one and returns false behind the last (or when a wait gave up); `done` gives its entry back.
struct Walk {
  const Shared& sm;
  uint32_t index = 0;
  Piece piece;
  __device__ __forceinline__ explicit Walk(const Shared& shared) : sm(shared) {}
  __device__ __forceinline__ bool next_of_warp() { return warp_wait(sm.bar(kPieceReady0 + index % kPieces), (index / kPieces) & 1, sm.abort_flag(), kLongWait) && read(); }
  __device__ __forceinline__ bool next_of_thread() { return mbar_wait(sm.bar(kPieceReady0 + index % kPieces), (index / kPieces) & 1, sm.abort_flag(), kLongWait) && read(); }
  __device__ __forceinline__ bool read() { piece = *sm.piece(index); return piece.first >= 0; }
  __device__ __forceinline__ void done() { mbar_arrive(sm.bar(kPieceDone0 + index % kPieces)); ++index; }  // one thread
  __device__ __forceinline__ void done_of_warp() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(sm.bar(kPieceDone0 + index % kPieces));
    ++index;
  }
};

// ---- copies ---------------------------------------------------------------------------------------------------------

template <int kWidth>
__device__ void copy_role(const Params& p, const Shared& sm) {
  using L = Layout<kWidth>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0, mended = 0;
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
    int pages = 0, next_pages = page_of(piece.first);  // of 32 chunks; of the next 32
    for (int chunk = piece.first; chunk < piece.last; ++chunk, ++count) {
      const int place = (chunk - piece.first) & 31;
      if (place == 0) {
        pages = next_pages;
        if (chunk + 32 < piece.last) next_pages = page_of(chunk + 32);
      }
      const int page = __shfl_sync(0xffffffffu, pages, place);
      const uint32_t stage = count % kStages, use = count / kStages, target = sm.base + stage * L::kTileBytes;
      if (use > 0 && !warp_wait(sm.bar(kFree0 + stage), (use - 1) & 1, abort_flag)) { given_up = true; break; }
      const bool legal = unsigned(page) < unsigned(p.blocks);
      const int valid = legal ? min(kChunk, piece.length - chunk * kChunk) : 0;
      const bool mend = valid < kChunk;
      const uint32_t bar = sm.bar(mend ? int(kMended) : int(kFull0 + stage));
      if (lane == 0) {
        *sm.live(stage) = valid;
        if (legal) {
          mbar_arrive_expect(bar, L::kTileBytes);
          const int row = page * p.page_rows + chunk * kChunk - over(chunk, p.by_page) * p.page_rows;
#pragma unroll
          for (int box = 0; box < L::kBoxes; ++box) copy_box(target + box * kBoxBytes, &p.cache, box * 64, row, bar);
        } else {
          report(p.status, SPARSE_MLA_STATUS_BAD_PAGE, int(piece.row / p.heads), chunk * kChunk);
        }
      }
      __syncwarp();
      if (mend) {
        if (legal && !warp_wait(bar, mended++ & 1, abort_flag)) { given_up = true; break; }
        for (int box = 0; box < LATENT_VALUES / 64; ++box)  // (the swizzle stays within a row)
          for (int at = valid * 128 + lane * 16; at < kBoxBytes; at += 512)
            *reinterpret_cast<uint4*>(sm.ptr + stage * L::kTileBytes + box * kBoxBytes + at) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(kFull0 + stage));
      }
    }
  }
  if (*abort_flag != 0) {  // nothing of this block may be written behind its end
    int never = 0;
    for (uint32_t i = count > kStages ? count - kStages : 0; i < count; ++i) mbar_wait(sm.bar(kFull0 + i % kStages), (i / kStages) & 1, &never);
    if (mended > 0) mbar_wait(sm.bar(kMended), (mended - 1) & 1, &never);
  }
}

// ---- queries --------------------------------------------------------------------------------------------------------

// Columns of 16 lanes (`taddr`'s lane field is the warp's lane base + 0 or + 16), see tmem_st_16x256b; eight columns.
__device__ __forceinline__ void tmem_st_8(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// A subpartition's 16 rows are shared by two warps: eight segments of 64 bytes each, and one of Q's last two. A thread loads 16 bytes of rows
// t / 4 and t / 4 + 8 of every segment; even words go to the low lanes and odd words to the high lanes as they are.
template <int kWidth>
__device__ void query_role(const Params& p, const Shared& sm, uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = sm.abort_flag();
  const int subpartition = warp & 3, part = (warp - kQueryWarp0) >> 2;
  const uint32_t lanes = uint32_t(subpartition * 32) << 16;
  constexpr int kOwn = kWidth / 64;  // segments of this warp
  uint32_t loads = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    if (piece.first == piece.last) continue;  // sees nothing
    uint4 words[2 * kOwn];
#pragma unroll
    for (int s = 0; s < kOwn; ++s) {
      const int segment = s < 8 ? part * 8 + s : 16 + part;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = subpartition * 16 + (lane >> 2) + 8 * k;
        words[2 * s + k] = make_uint4(0, 0, 0, 0);
        if (row < piece.rows) words[2 * s + k] = *reinterpret_cast<const uint4*>(p.q + (piece.row + row) * (kWidth * 2) + segment * 64 + (lane & 3) * 16);
      }
    }
    if (loads > 0 && !warp_wait(sm.bar(kQFree), (loads - 1) & 1, abort_flag, kLongWait)) return;
    tc_fence_after_sync();
#pragma unroll
    for (int s = 0; s < kOwn; ++s) {
      const uint32_t at = tmem + lanes + (s < 8 ? kColumnsQ + (part * 8 + s) * 8 : kColumnsQRest + part * 8);
      const uint4 a = words[2 * s], b = words[2 * s + 1];
      tmem_st_8(at, a.x, a.z, b.x, b.z);
      tmem_st_8(at + kHighLanes, a.y, a.w, b.y, b.w);
    }
    tmem_wait_st();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.bar(kQFull));
    ++loads;
  }
}

// ---- products (one thread each) --------------------------------------------------------------------------------------

template <int kFormat> constexpr uint32_t kIdescScores = idesc_f16(128, kChunk, kFormat, 0, 0) | kSparseA;
template <int kFormat> constexpr uint32_t kIdescValues = idesc_f16(64, 256, kFormat, 0, 1);  // issued as .ws

// A tile's boxes of 64 features are kBox bytes apart, its groups of eight rows kGroup.
template <int kFormat, int kSteps, int kBox, int K = 0>
__device__ __forceinline__ void issue_scores(uint32_t tmem, uint64_t x_desc) {
  if constexpr (K < kSteps) {
    constexpr uint32_t offset = (K >> 1) * kBox + (K & 1) * 64;
    constexpr uint32_t q = K < 16 ? kColumnsQ + K * 8 : kColumnsQRest + (K - 16) * 8;
    mma_sparse_ts_c<K != 0>(tmem + kColumnsScores, tmem + q, x_desc + (offset >> 4), tmem + kColumnsPlaces, kIdescScores<kFormat>);
    issue_scores<kFormat, kSteps, kBox, K + 1>(tmem, x_desc);
  }
}
// Steps I to kEnd - 1 of the chunk's, two for every 16 rows.
template <int kFormat, int kBox, int kGroup, bool kFirst, int kEnd, int I>
__device__ __forceinline__ void issue_values(uint32_t tmem, uint64_t p_desc, uint64_t x_desc) {
  if constexpr (I < kEnd) {
    constexpr int half = I % 2, k = I / 2;
    constexpr uint32_t offset = half * 4 * kBox + k * 2 * kGroup;
    mma_ws_ss_c<!(kFirst && k == 0)>(tmem + half * 128, p_desc + ((k * 32) >> 4), x_desc + (offset >> 4), kIdescValues<kFormat>);
    issue_values<kFormat, kBox, kGroup, kFirst, kEnd, I + 1>(tmem, p_desc, x_desc);
  }
}

template <int kFormat, int kWidth, int kBox, int kGroup>
__device__ void score_role(const Shared& sm, uint32_t tmem) {
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0, loads = 0;
  Walk walk(sm);
  if (!mbar_wait(sm.bar(kPlaces), 0, abort_flag)) return;
  for (; walk.next_of_thread(); walk.done()) {
    const int chunks = walk.piece.last - walk.piece.first;
    if (chunks == 0) continue;
    if (!mbar_wait(sm.bar(kQFull), loads++ & 1, abort_flag)) return;
    for (int i = 0; i < chunks; ++i, ++count) {
      const uint32_t stage = count % kStages;
      if (!mbar_wait(sm.bar(kFull0 + stage), (count / kStages) & 1, abort_flag)) return;
      if (!mbar_wait(sm.bar(kScoresFree), (count & 1) ^ 1, abort_flag)) return;
      tc_fence_after_sync();
      issue_scores<kFormat, kWidth / 32, kBox>(tmem, smem_desc_sw128(sm.base + stage * Layout<kWidth>::kTileBytes, 16, kGroup));
      mma_commit(sm.bar(kScoresFull));
    }
    mma_commit(sm.bar(kQFree));
  }
}

// kHalves: says so when the first half of the chunk's rows have been used.
template <int kFormat, int kWidth, int kBox, int kGroup, bool kHalves>
__device__ void value_role(const Shared& sm, uint32_t tmem) {
  volatile int* abort_flag = sm.abort_flag();
  uint32_t count = 0;
  Walk walk(sm);
  const uint64_t p_desc = smem_desc_sw128(sm.base + Layout<kWidth>::kSmemP, 16, 1024);
  for (; walk.next_of_thread(); walk.done()) {
    const int chunks = walk.piece.last - walk.piece.first;
    for (int i = 0; i < chunks; ++i, ++count) {
      const uint32_t stage = count % kStages;
      if (!mbar_wait(sm.bar(kWeightsFull), count & 1, abort_flag)) return;
      tc_fence_after_sync();
      const uint64_t x_desc = smem_desc_sw128(sm.base + stage * Layout<kWidth>::kTileBytes, kBox, kGroup);
      constexpr int kSteps = 2 * (kChunk / 16);
      if constexpr (kHalves) {
        if (i == 0) issue_values<kFormat, kBox, kGroup, true, kSteps / 2, 0>(tmem, p_desc, x_desc);
        else issue_values<kFormat, kBox, kGroup, false, kSteps / 2, 0>(tmem, p_desc, x_desc);
        mma_commit(sm.bar(kFreeHalf0 + stage));
        issue_values<kFormat, kBox, kGroup, false, kSteps, kSteps / 2>(tmem, p_desc, x_desc);
      } else {
        if (i == 0) issue_values<kFormat, kBox, kGroup, true, kSteps, 0>(tmem, p_desc, x_desc);
        else issue_values<kFormat, kBox, kGroup, false, kSteps, 0>(tmem, p_desc, x_desc);
      }
      mma_commit(sm.bar(kWeightsFree));
      mma_commit(sm.bar(kFree0 + stage));
    }
  }
}

// ---- softmax ----------------------------------------------------------------------------------------------------------

// A row's reference (log2) starts kFirst below the maximum of its first scores and moves when others exceed it by more than kRoom, to kStep below
// them. Weights are rounded to the storage type for the second product; in IEEE half they fit up to 65504, so that the accumulator is
// rarely rescaled. What counts below the greatest is off there by at most 2^-25 of the unit, which is 2^-31 of the greatest: 128 K of those are
// 2^-14. (With the first reference at the maximum itself they were 2^-8, and keys 25 binades below a dominant first one were lost altogether. bfloat16 has
// the range for that.) The lower the first reference, the sooner it moves: scores of a deviation of 3, half, 64 x 1 at 8K 131.9 us, 128.6 with 0, 132.3 with 8;
// of 1 the same with all.
constexpr float kRoom = 15.9f, kStep = 8.f;
template <int kFormat> constexpr float kFirst = kFormat == 1 ? 0.f : 6.f;
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 1 / denominator and the log (log2) of it, from a row's reference and sum and its sink (log2; -infinity: none).
__device__ __forceinline__ float inverse_of(float reference, float sum, float sink, float* log_sum) {
  const float own = sum == 0.f ? -INFINITY : reference + log2f(sum);
  if (sink == -INFINITY) {
    *log_sum = own;
    return sum == 0.f ? 0.f : 1.f / sum;
  }
  const float top = fmaxf(own, sink), share = exp2f(own - top), total = share + exp2f(sink - top);
  *log_sum = top + log2f(total);
  return sum == 0.f ? 0.f : share / (total * sum);
}

template <int kFormat, int kWidth, bool kHeld8>
__device__ void softmax_role(const Params& p, const Shared& sm, uint32_t tmem) {
  using L = Layout<kWidth>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4;
  volatile int* abort_flag = sm.abort_flag();
  const uint32_t lanes = uint32_t(warp * 32) << 16, scores = tmem + kColumnsScores + lanes;
  // This thread works out weights of row `row`, of keys 32 half .. + 31 of a chunk; the accumulator's lane that it reads belongs to another row.
  const int row = warp * 16 + (lane & 15), o_row = (warp & 1) * 32 + lane, o_feature = (warp >> 1) * 128;
  float* alphas = reinterpret_cast<float*>(sm.ptr + L::kSmemAlpha);
  float* inverses = reinterpret_cast<float*>(sm.ptr + L::kSmemInverse);
  unsigned char* weights = sm.ptr + L::kSmemP;
  {
    uint32_t columns[16];  // which pairs a lane of Q holds: numbers 0 and 1 of every four features, or 2 and 3
#pragma unroll
    for (int e = 0; e < 16; ++e) columns[e] = half ? 0xeeeeeeeeu : 0x44444444u;
    tmem_st16(tmem + kColumnsPlaces + lanes, columns);
    tmem_wait_st();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.bar(kPlaces));
  }
  // The four warps meet once a chunk. One whose wait gave up says so there, and all leave behind it.
  bool failed = false;
  constexpr uint32_t kGivenUp = 32;
  auto meet = [&](bool flag) { return named_barrier_count(1, 32 * kSoftmaxWarps, failed || (flag && lane == 0)); };
  uint32_t count = 0;
  Walk walk(sm);
  for (; walk.next_of_warp(); walk.done_of_warp()) {
    const Piece& piece = walk.piece;
    const int chunks = piece.last - piece.first;
    const int end = row < piece.rows ? piece.base + over(piece.head + row, p.by_heads) + piece.token : INT32_MAX;  // this row sees keys below
    const int warp_end = __reduce_min_sync(0xffffffffu, end);
    float reference = -INFINITY, sum = 0.f;
    for (int i = 0; i < chunks; ++i, ++count) {
      const uint32_t stage = count % kStages;
      // (the tile has landed when its scores are there; this wait makes what was written about it visible)
      if (!warp_wait(sm.bar(kScoresFull), count & 1, abort_flag) || !warp_wait(sm.bar(kFull0 + stage), (count / kStages) & 1, abort_flag)) { failed = true; meet(true); return; }
      tc_fence_after_sync();
      const int key = (piece.first + i) * kChunk;
      int live = kHeld8 ? *sm.marked(stage) : *sm.live(stage);
      float2 s[16];
      {
        // Both partial sums of a score come straight to the thread that owns it.
        uint32_t low_a[16], low_b[16], high_a[16], high_b[16];
        tmem_ld16_halves<32>(scores, low_a);
        tmem_ld16_halves<32>(scores + 16, low_b);
        tmem_ld16_halves<32>(scores + kHighLanes, high_a);
        tmem_ld16_halves<32>(scores + kHighLanes + 16, high_b);
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(kScoresFree));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[e] = add2(make_float2(__uint_as_float(low_a[2 * e]), __uint_as_float(low_a[2 * e + 1])),
                      make_float2(__uint_as_float(high_a[2 * e]), __uint_as_float(high_a[2 * e + 1])));
          s[8 + e] = add2(make_float2(__uint_as_float(low_b[2 * e]), __uint_as_float(low_b[2 * e + 1])),
                          make_float2(__uint_as_float(high_b[2 * e]), __uint_as_float(high_b[2 * e + 1])));
        }
      }
      if (live < kChunk || key + kChunk > warp_end) {
        if (kHeld8 && live < 0) {  // keys whose scales are NaN: their values are zeros here
          live += kSpoilt;
          const uint32_t spoilt = *sm.spoilt(stage, half);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (spoilt >> 2 * e & 1) s[e].x = __uint_as_float(0x7fc00000u);
            if (spoilt >> 2 * e & 2) s[e].y = __uint_as_float(0x7fc00000u);
          }
        }
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
      const float own = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale_log2;  // scale > 0
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
      float* factors = alphas + (count & 1) * kRows;
      if (half == 0) factors[row] = alpha;
      const float shift = reference == -INFINITY ? 0.f : -reference;
      const float2 scale = make_float2(p.scale_log2, p.scale_log2), shifts = make_float2(shift, shift);
      float2 sum_a = make_float2(0.f, 0.f), sum_b = sum_a;
      uint4 packed[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t words[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int e = 4 * u + w;
          float2 weight = fma2(s[e], scale, shifts);
          weight.x = exp2f(weight.x);
          weight.y = exp2f(weight.y);
          if (e & 1) sum_b = add2(sum_b, weight); else sum_a = add2(sum_a, weight);
          words[w] = pack2<kFormat>(weight.x, weight.y);
        }
        packed[u] = make_uint4(words[0], words[1], words[2], words[3]);
      }
      sum = sum * alpha + ((sum_a.x + sum_a.y) + (sum_b.x + sum_b.y));
      // The product of the chunk before has ended: its weights may be overwritten, the accumulator rescaled.
      if (count > 0 && !warp_wait(sm.bar(kWeightsFree), (count - 1) & 1, abort_flag)) { failed = true; meet(true); return; }
#pragma unroll
      for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4*>(weights + row * 128 + (((half * 4 + u) ^ (row & 7)) << 4)) = packed[u];
      const uint32_t met = meet(look && i > 0);
      if (met >= kGivenUp) return;
      if (met != 0) {
        tc_fence_after_sync();
        const float o_alpha = factors[o_row];
#pragma unroll 1
        for (int c = 0; c < 256; c += 32) {
          uint32_t o[32];
          tmem_ld32(tmem + c + lanes, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * o_alpha);
          tmem_st32(tmem + c + lanes, o);
        }
        tmem_wait_st();
      }
      fence_proxy_async();  // the product reads the weights through the async proxy
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(kWeightsFull));
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    // ---- output
    if (chunks > 0) {
      if (!warp_wait(sm.bar(kWeightsFree), (count - 1) & 1, abort_flag)) { failed = true; meet(true); return; }
      tc_fence_after_sync();
    }
    if (piece.slot >= 0) {  // a part of a tile: sums as they are
      if (half == 0 && row < piece.rows) p.statistics[size_t(piece.slot) * kRows + row] = part_statistics(reference, sum);
      float* sums = p.sums + size_t(piece.slot) * kSlotFloats + sums_place(o_row, o_feature);
#pragma unroll 1
      for (int c = 0; c < 256; c += 64) {
        uint32_t o[64];
        tmem_ld32(tmem + c + lanes, o);
        tmem_ld32(tmem + c + 32 + lanes, o + 32);
        tmem_wait_ld();
        if (o_row < piece.rows) {
#pragma unroll
          for (int e = 0; e < 64; e += 8) store_sector(sums + (c + e) * 32, o + e);
        }
      }
      continue;
    }
    float log_sum;
    const float sink = p.sinks != nullptr && row < piece.rows ? p.sinks[(piece.head + row) % p.heads] * kLog2E : -INFINITY;
    const float inverse = inverse_of(reference, sum, sink, &log_sum);
    if (half == 0) {
      inverses[row] = inverse;
      if (p.lse != nullptr && row < piece.rows) p.lse[piece.row + row] = log_sum * kLn2;
    }
    if (meet(false) != 0) return;
    const float o_inverse = inverses[o_row];
    // 32 rows x 64 bytes per warp and pass, through the warp's quarter of the weights' tile.
    unsigned char* staged = weights + warp * 2048;
#pragma unroll 1
    for (int c = 0; c < 256; c += 32) {
      uint32_t o[32];
      if (chunks > 0) {
        tmem_ld32(tmem + c + lanes, o);
        tmem_wait_ld();
      }
#pragma unroll
      for (int unit = 0; unit < 4; ++unit) {
        uint32_t words[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          words[k] = chunks == 0 || o_inverse == 0.f ? 0u : pack2<kFormat>(__uint_as_float(o[unit * 8 + 2 * k]) * o_inverse, __uint_as_float(o[unit * 8 + 2 * k + 1]) * o_inverse);
        *reinterpret_cast<uint4*>(staged + lane * 64 + ((unit ^ ((lane >> 1) & 3)) << 4)) = make_uint4(words[0], words[1], words[2], words[3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2), unit = lane & 3, target = (warp & 1) * 32 + r;
        const uint4 v = *reinterpret_cast<const uint4*>(staged + r * 64 + ((unit ^ ((r >> 1) & 3)) << 4));
        if (target < piece.rows)
          *reinterpret_cast<uint4*>(p.out + ((piece.row + target) * LATENT_VALUES + (c >> 7) * 256 + o_feature + (c & 127) + unit * 8) * 2) = v;
      }
      __syncwarp();
    }
    if (meet(false) != 0) return;  // the inverses and the weights' tile are free again
  }
  if (*abort_flag != 0) failed = true;
  meet(false);  // with a warp that has given up since the last time
}

}  // namespace absorbed
}  // namespace latent

#include "latent_held8.cuh"
#include "latent_turned8.cuh"

namespace latent {
namespace absorbed {

// ---- kernels and launch ------------------------------------------------------------------------------------------------

// kHeld8: rows in 8 bits; the warps from number 6 on have other roles then, see latent_held8.cuh.
template <int kFormat, int kWidth, bool kHeld8>
__global__ void __launch_bounds__(kHeld8 ? kThreads8 : kThreads, 1) attention_kernel(const __grid_constant__ Params p) {
  using L = Layout<kWidth>;
  constexpr int kOwnThreads = kHeld8 ? kThreads8 : kThreads, kOwnQueryWarps = kHeld8 ? kQueryWarps8 : kQueryWarps;
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
      if (i >= kPieceDone0 && i < kPieceDone0 + kPieces) arrivals = kSoftmaxWarps + 3 + (kHeld8 ? kConvertWarps : 0) + kOwnQueryWarps;
      else if (i == kQFull) arrivals = kOwnQueryWarps;
      else if (kHeld8 && i < kFull0 + kStages) arrivals = kConvertWarps;
      else if (i == kScoresFree || i == kWeightsFull || i == kPlaces) arrivals = kSoftmaxWarps;
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
    borders = plan_block<kOwnThreads / 32>(p, sm.scan(), &place);
    fence_proxy_async();  // the plan's scratch is the first tile's memory
    __syncthreads();
  }
  auto issue = [&]() {
    if (elect_one()) {
      constexpr int kBox = kHeld8 ? 1024 : kBoxBytes, kGroup = kHeld8 ? kGroupBytes<kWidth> : 1024;
      if (warp == kScoreWarp) score_role<kFormat, kWidth, kBox, kGroup>(sm, tmem);
      else value_role<kFormat, kWidth, kBox, kGroup, kHeld8>(sm, tmem);
      if (*sm.abort_flag() != 0) wait_for_products(sm.bar(warp == kScoreWarp ? kGivenUp0 : kGivenUp1));
    }
    __syncwarp();
  };
  auto plan = [&]() {
    if (p.batches <= 32) borders = plan_block<1>(p, nullptr, &place);
    plan_role(p, sm, borders, place);
  };
  if constexpr (kHeld8) {
    if (warp < kSoftmaxWarps) {
      take_128_registers();
      softmax_role<kFormat, kWidth, kHeld8>(p, sm, tmem);
    } else if (warp < kConvertWarp0) {
      keep_64_registers();
      if (warp == kScoreWarp || warp == kValueWarp) issue();
      else if (warp == kCopyWarp) copy_role8<kWidth>(p, sm);
      else if (warp == kPlanWarp) plan();
      else if (warp >= kQueryWarp0) query_role8<kWidth>(p, sm, tmem);
    } else {
      take_112_registers();
      convert_role<kFormat, kWidth>(p, sm);
    }
  } else {
    if (warp < kSoftmaxWarps) softmax_role<kFormat, kWidth, kHeld8>(p, sm, tmem);
    else if (warp == kScoreWarp || warp == kValueWarp) issue();
    else if (warp == kCopyWarp) copy_role<kWidth>(p, sm);
    else if (warp == kPlanWarp) plan();
    else query_role<kWidth>(p, sm, tmem);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && *sm.abort_flag() != 0) report(p.status, SPARSE_MLA_STATUS_WAIT_EXPIRED, blockIdx.x, 0);
  if (warp == kScoreWarp) tmem_dealloc(tmem, 512);
}

// Tiles that several blocks worked on. Every block makes the list of them, with what there is to do for each: 32 features of eight rows by one to
// eight warps of a block, as many as bring all parts with one round of loads if there are blocks enough for that. Sums are added in the order of
// the parts (of the warps' shares), whatever block does it. Bound by latency: the list; statistics and the first round of sums together; the others.
// (8 requests of 8192 keys, one token, 64 heads, 18 parts each: 4.0 us, and 8.7 with eight warps for every half row and statistics in front of the sums.)
constexpr int kMostBlocks = 256, kUnits = LATENT_VALUES / kUnitFeatures;

// kTurned: a slot's sums lie row by row (latent_turned8.cuh).
template <int kFormat, bool kTurned>
__global__ void __launch_bounds__(kCombineThreads, 2) combine_kernel(const __grid_constant__ Params p, int blocks) {
  struct Tile {
    int64_t row;
    int rows, head, block, parts, warps, items;  // `items` for a block: with those in front of it
  };
  __shared__ int wishes[kCombineWarps], ends[kCombineWarps];
  __shared__ Tile list[kMostBlocks];
  __shared__ Shares shared;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_predecessor();
  let_successor_start();
  {
    const int own = threadIdx.x;
    Record record = {0, 0, 0, -1, {0, 0, 0}};
    if (own < blocks) record = p.records[own];
    const int parts = record.last >= 0 ? record.last - own + 1 : 0;
    int warps = warps_for(parts);
    const int wish = __reduce_add_sync(0xffffffffu, parts == 0 ? 0 : (record.rows + kUnitRows - 1) / kUnitRows * kUnits * warps);
    if (lane == 0) wishes[warp] = wish;
    __syncthreads();
    int wanted = 0;
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) wanted += wishes[w];
    for (; wanted > int(gridDim.x) * kCombineWarps; wanted >>= 1) warps = max(1, warps >> 1);
    const int items = parts == 0 ? 0 : (record.rows + kUnitRows - 1) / kUnitRows * kUnits * warps / kCombineWarps;
    int packed = items << 8 | (parts > 0);  // both sums at once: items below 2^16, tiles below 2^8
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, packed, d);
      if (lane >= d) packed += other;
    }
    if (lane == 31) ends[warp] = packed;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w)
      if (w < warp) packed += ends[w];
    if (parts > 0) list[(packed & 255) - 1] = {record.row, record.rows, record.head, own, parts, warps, packed >> 8};
    __syncthreads();
  }
  int items = 0;
#pragma unroll
  for (int w = 0; w < kCombineWarps; ++w) items += ends[w] >> 8;
  int index = 0;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    while (list[index].items <= item) ++index;
    const Tile tile = list[index];
    const int place = item - (index > 0 ? list[index - 1].items : 0), warps = tile.warps;
    const int unit = (place * kCombineWarps + warp) / warps;
    const int rows = unit / kUnits * kUnitRows, segment = unit % kUnits;
    auto feature_of = [&](int lane) { return (segment >> 3) * 256 + (segment & 1) * 128 + (segment >> 1 & 3) * 32 + (lane >> 3) * 8; };
    auto slot_of = [&](int part) { return size_t(part == 0 ? 2 * tile.block + 1 : 2 * (tile.block + part)); };
    join_parts<kFormat>(
        shared, warps, tile.parts, rows, tile.rows,
        [&](int part, int row) { return p.sums + slot_of(part) * kSlotFloats + (kTurned ? row * LATENT_VALUES + feature_of(lane) : sums_place(row, feature_of(lane))); },
        [&](int part, int row) { return p.statistics + slot_of(part) * kRows + row; },
        [&](int row, int owner) { return p.out + ((tile.row + row) * LATENT_VALUES + feature_of(owner)) * 2; },
        [&](int row, float reference, float sum, bool first_of_row) {  // what the row's sums are multiplied with
          float log_sum;
          const float sink = p.sinks != nullptr ? p.sinks[(tile.head + row) % p.heads] * kLog2E : -INFINITY;
          const float inverse = inverse_of(reference, sum, sink, &log_sum);
          if (p.lse != nullptr && first_of_row && segment == 0) p.lse[tile.row + row] = log_sum * kLn2;
          return inverse;
        });
  }
}

// One block per SM; no more than `combine_kernel` has room for.
int grid() { const int count = multiprocessors(); return count < kMostBlocks ? count : kMostBlocks - 1; }

// How a call is worked out: rows in 16 bits; rows in 8 bits, widened to 16-bit tiles; rows in 8 bits, the other way round (latent_turned8.cuh).
enum Form { kWide, kHeld, kTurnedRound };

template <int kFormat, int kWidth, int kForm>
int launch(const Params& p, int blocks, cudaStream_t stream) {
  constexpr bool kHeld8 = kForm != kWide, kTurned = kForm == kTurnedRound;
  static_assert(!kTurned || kFormat == 1, "a query of half has more bits than two numbers of 8");
  void (*kernel)(Params) = nullptr;
  int shared_bytes = 0, threads = 0;
  if constexpr (kTurned) {
    kernel = turned::attention_kernel<kWidth>;
    shared_bytes = turned::Layout<kWidth>::kSmemBytes;
    threads = turned::kThreads;
  } else {
    kernel = attention_kernel<kFormat, kWidth, kHeld8>;
    shared_bytes = Layout<kWidth>::kSmemBytes;
    threads = kHeld8 ? kThreads8 : kThreads;
  }
  static bool configured[64] = {false};  // a per-device setting: plain words written with the same value by whoever gets there first
  int device = 0;
  if (const cudaError_t error = cudaGetDevice(&device)) return int(error);
  if (device < 0 || device >= 64) return -1;
  if (!configured[device]) {
    if (const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes)) return int(error);
    configured[device] = true;
  }
  if (const cudaError_t error = launch_overlapped(kernel, blocks, threads, shared_bytes, stream, p)) return int(error);
  cudaLaunchAttribute overlap = {};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(blocks) * 2);
  config.blockDim = dim3(kCombineThreads);
  config.stream = stream;
  config.attrs = &overlap;
  config.numAttrs = 1;
  return int(cudaLaunchKernelEx(&config, combine_kernel<kFormat, kTurned>, p, blocks));
}

}  // namespace absorbed
}  // namespace latent

extern "C" {

int workspace_size_latent_attention(uint64_t* bytes) {
  using namespace latent;
  if (bytes == nullptr) return -1;
  *bytes = absorbed::workspace_bytes(absorbed::grid());
  return 0;
}

}  // extern "C"

namespace latent {
namespace absorbed {
namespace {

// From so many chunks to a block on bfloat16 queries over rows in 8 bits go the other way round, whose start takes 6 us longer and whose chunks 8 per cent less. The other way
// round / not, us, of 64 heads (chunks): one token of 8K rows (0.9) 23.8 / 18.4; 16 of them (14) 42.5 / 41.3; 64 at 2K (14) 48.9 / 47.1; 24 at 8K (21) 53.7 / 55.1;
// 8 x 6 at 4K (21) 52.8 / 49.4; 32 at 8K (28) 63.4 / 66.7; 16 x 6 at 4K (42) 84.4 / 85.4; 64 at 8K (55) 102.9 / 117.0; 500 tokens of 16 heads at 8K (108) 165 / 175. (The
// host knows the table's width only, which is the longest that requests may be: hence not from 24 on. Short requests under a wide table pay for it: 8 at 2K under one for 128K 26.5 / 19.1, 32 at 2K
// 33.9 / 28.5, 8 at 8K 34.0 / 27.7, 64 at 2K 48.7 / 47.4.)
constexpr int64_t kTurnedChunks = 32;

template <bool kHeld8>
int launch_call(void* stream, const latent_attention_call& c, const uint8_t* scales, int64_t block_rows) {
  if ((c.type != LATENT_F16 && c.type != LATENT_BF16) || (c.width != 512 && c.width != 576) || !scale_fits(c.scale)) return -1;
  if (c.batches < 0 || c.batches > INT32_MAX / 2 || c.tokens < 0 || c.heads < 1 || c.tokens > (int64_t(1) << 30) / c.heads) return -1;
  if (c.pages < 0 || c.blocks < 0 || c.page_rows < 64 || c.page_rows % 64 != 0 || c.pages > (INT32_MAX - 128) / c.page_rows || c.blocks > INT32_MAX / c.page_rows) return -1;
  if (!aligned(c.q) || !aligned(c.cache) || !aligned(c.out)) return -1;
  if (kHeld8 && (block_rows < 1 || block_rows > 64 || (block_rows & (block_rows - 1)) != 0)) return -1;
  if (c.tokens == 0 || c.batches == 0) return 0;
  if (c.workspace == nullptr || reinterpret_cast<uintptr_t>(c.workspace) % 32 != 0 || c.status == nullptr) return -1;
  const int blocks = grid();
  Params p = {};
  if constexpr (kHeld8) {
    const int64_t rows = c.blocks > 0 ? c.blocks * c.page_rows : 1;  // (without pages nothing is copied)
    const void* base = c.blocks > 0 ? c.cache : c.q;
    if (c.type == LATENT_BF16) {
      if (const int e = turned::encode_map8(&p.cache, base, c.width, rows, 128)) return e;
      if (const int e = turned::encode_map8(&p.rest, base, c.width, rows, 64)) return e;
    }
    p.held = static_cast<const char*>(c.cache);
    p.scales = scales;
    while ((int64_t(1) << p.block_shift) < block_rows) ++p.block_shift;
  } else {
    // (without pages nothing is copied)
    const int64_t sizes[2] = {c.width, c.blocks > 0 ? c.blocks * c.page_rows : 1}, strides[1] = {c.width};
    if (const int e = sm100::encode_map(&p.cache, c.type, 2, c.blocks > 0 ? c.cache : c.q, sizes, strides, 1, kChunk)) return e;
  }
  char* workspace = static_cast<char*>(c.workspace);
  p.q = static_cast<const char*>(c.q);
  p.table = c.block_table;
  p.cu = c.cu_seqlens_q;
  p.lengths = c.seqused_kv;
  p.sinks = c.sinks;
  p.out = static_cast<char*>(c.out);
  p.lse = c.lse;
  p.records = reinterpret_cast<Record*>(workspace);
  p.statistics = reinterpret_cast<float2*>(workspace + statistics_offset(blocks));
  p.sums = reinterpret_cast<float*>(workspace + sums_offset(blocks));
  p.status = c.status;
  p.batches = int32_t(c.batches);
  p.tokens = int32_t(c.tokens);
  p.heads = int32_t(c.heads);
  p.by_heads = divisor_of(p.heads);
  p.tile_tokens = kRows / p.heads + 1;
  p.pages = int32_t(c.pages);
  p.blocks = int32_t(c.blocks);
  p.page_rows = int32_t(c.page_rows);
  p.by_page = divisor_of(p.page_rows / kChunk);
  p.scale_log2 = float(c.scale * 1.4426950408889634);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  constexpr Form kForm = kHeld8 ? kHeld : kWide;
  if constexpr (kHeld8) {
    // Chunks to a block, if requests are as long as the table.
    const int64_t tiles = std::max((c.tokens * c.heads + kRows - 1) / kRows, std::min(c.batches, c.tokens));
    const int64_t chunks = tiles * std::min(c.pages, c.blocks) * (c.page_rows / kChunk) / blocks;
    if (c.type == LATENT_BF16 && chunks >= kTurnedChunks) return c.width == 576 ? launch<1, 576, kTurnedRound>(p, blocks, s) : launch<1, 512, kTurnedRound>(p, blocks, s);
  }
  if (c.type == LATENT_BF16) return c.width == 576 ? launch<1, 576, kForm>(p, blocks, s) : launch<1, 512, kForm>(p, blocks, s);
  return c.width == 576 ? launch<0, 576, kForm>(p, blocks, s) : launch<0, 512, kForm>(p, blocks, s);
}

}  // namespace
}  // namespace absorbed
}  // namespace latent

extern "C" {

int launch_latent_attention(void* stream, const latent_attention_call* call) { return call == nullptr ? -1 : latent::absorbed::launch_call<false>(stream, *call, nullptr, 0); }

int launch_latent_attention8(void* stream, const latent_attention8_call* call) {
  return call == nullptr ? -1 : latent::absorbed::launch_call<true>(stream, call->attention, call->scales, call->block_rows);
}

}  // extern "C"
