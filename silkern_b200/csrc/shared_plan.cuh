// Attention behind shared prefixes: its arguments, its workspace, and how the
// work is laid over the GPU.
//
// A segment is a group's prefix with all of the group's queries, or a
// sequence's own tokens with its own. Its rows are its (query, head) pairs of
// one cache head, token by token, in blocks of 256; an item is one block of rows
// over the segment's keys, for every cache head. Items' tiles of 128 keys, item
// by item and head by head, are one line of units of time (with some more for
// each item and head, for its start and end), which the grid's CTAs cut into
// equal parts, by the lengths that stand on the device. A tile is the CTA's in
// whose part its first unit lies. A CTA's share of an item and head is a
// fragment, whose outputs and log-sum-exps go to the workspace; a second kernel
// joins each row's.
#pragma once

#include "paged.cuh"

namespace silkern {

constexpr int kSharedTile = 128;   // keys
constexpr int kSlotRows = 128;     // rows of a softmax warpgroup
constexpr int kBlockRows = 2 * kSlotRows;
constexpr int kLeastUnits = 16;    // of a CTA: a tile of every sort at least
constexpr int kMostCtas = 148;     // one to an SM

struct SharedHeader {
  int64_t units;  // of all items and heads
  int64_t share;  // of a CTA
  int32_t items;
  int32_t failed;  // a wait ran out
};

struct __align__(16) SharedItem {
  int64_t begin;      // units of the items before it, of one cache head
  int32_t tiles;
  int32_t key_begin;  // rank-local keys from here, at a multiple of 16,
  int32_t key_first;  // of which those from here
  int32_t key_end;    // to here count
  int32_t table_row;
  int32_t token;      // the segment's first
  int32_t row, rows;  // rows [row, row + rows) of the segment
  int32_t seq, seqs;  // its sequences
  int32_t extra;      // rows of one cache head that other items' second copies take before it
  int32_t prefix;     // 1: a group's, 0: a sequence's own
  int32_t pad[2];
};
static_assert(sizeof(SharedItem) == 64, "read in four parts");

// Where things lie in the workspace, in bytes from its start.
struct SharedLayout {
  int64_t limits;    // (groups,): the longest length, where they are too many for the plan's shared memory
  int64_t first;     // (groups,): a prefix's first item; -1: none
  int64_t records;   // (sequences,): its first item (-1: none) and token, its group's first item and token
  int64_t items;
  int64_t most_items;
  int64_t lse;       // of the partial rows, base 2
  int64_t out;       // (partial rows, dim) float32
  int64_t starts;    // partial rows before those of CTAs' first fragments
  int64_t copies;    // and before the second copies
  int64_t bytes;
};

struct SharedArgs {
  PagedCache cache;
  const void* q;
  int64_t q_row, q_head;
  void* out;
  int64_t out_row, out_head;
  bool out_wide;
  float* lse;
  int32_t* status;
  uint8_t* work;
  SharedLayout at;
  int64_t wait_cycles;
  float scale_log2;  // |softmax_scale| * log2(e)
  float q_sign;
  int32_t rows, heads, heads_per_kv;
  FastDiv per_kv;  // by heads_per_kv
  int32_t sequences, groups;
  bool runs;  // pages hold whole runs of 16 keys
  const int32_t* cu_tokens;
  const int32_t* lengths;
  const int32_t* req_ids;
  const int32_t* cu_groups;
  const int32_t* prefixes;
  const int32_t* table;
  int64_t table_rows;
  uint32_t table_width;
  Ownership own;

  __device__ __forceinline__ SharedHeader* header() const { return reinterpret_cast<SharedHeader*>(work); }
  __device__ __forceinline__ SharedItem* item(int32_t i) const { return reinterpret_cast<SharedItem*>(work + at.items) + i; }
  __device__ __forceinline__ int32_t* first() const { return reinterpret_cast<int32_t*>(work + at.first); }
  __device__ __forceinline__ int4* records() const { return reinterpret_cast<int4*>(work + at.records); }
  __device__ __forceinline__ int32_t* limits() const { return reinterpret_cast<int32_t*>(work + at.limits); }
  __device__ __forceinline__ float* part_lse() const { return reinterpret_cast<float*>(work + at.lse); }
  __device__ __forceinline__ float* part_out() const { return reinterpret_cast<float*>(work + at.out); }
  // A sequence's first token, within q.
  __device__ __forceinline__ int32_t cu(int32_t seq) const { return min(max(load_int(cu_tokens + seq), 0), rows); }
  __device__ __forceinline__ int32_t cut(int32_t group) const { return min(max(load_int(cu_groups + group), 0), sequences); }
  // How many rank-local keys the positions below `n` have.
  __device__ __forceinline__ int32_t keys_below(int32_t n) const {
    return n <= 0 ? 0 : static_cast<int32_t>(own.owned_before(static_cast<uint32_t>(n)));
  }
};

// Units of a tile, and of an item's start and end, by its rows: about 500 cycles
// each, as measured with 128 columns; those of 64 are cut by the same ones. Up to
// 128 rows the slots take turns with the tiles, and one's start hides behind the
// other's tiles.
__device__ __forceinline__ int32_t units_of_tile(int32_t rows) { return rows <= kSlotRows ? 6 : 8; }
__device__ __forceinline__ int32_t units_of_start(int32_t rows) { return rows <= kSlotRows ? 19 : 46; }
__device__ __forceinline__ int64_t units_of(int32_t tiles, int32_t rows) {
  return tiles > 0 ? units_of_start(rows) + static_cast<int64_t>(tiles) * units_of_tile(rows) : 0;
}

// The last i in [0, n) with at(i) <= x, for at that ascends from at(0) <= x.
template <typename F>
__device__ __forceinline__ int32_t last_at_most(int32_t n, int64_t x, F at) {
  int32_t low = 0, high = n;
  while (high - low > 1) {
    const int32_t mid = low + (high - low) / 2;
    if (at(mid) <= x) low = mid; else high = mid;
  }
  return low;
}
// The same by a whole warp, 32 places a step.
template <typename F>
__device__ __forceinline__ int32_t warp_last_at_most(int32_t n, int64_t x, F at) {
  const int32_t lane = threadIdx.x & 31;
  int32_t low = 0, high = n;
  while (high - low > 1) {
    const int32_t step = (high - low + 31) / 32, i = low + lane * step;
    const uint32_t hits = __ballot_sync(kAllLanes, i < high && at(i) <= x);
    const int32_t last = hits == 0 ? 0 : 31 - __clz(hits);
    low += last * step;
    high = min(high, low + step);
  }
  return low;
}

int launch_shared_dim64(const SharedArgs& a, bool half, unsigned grid, cudaStream_t stream);
int launch_shared_dim128(const SharedArgs& a, bool half, unsigned grid, cudaStream_t stream);

}  // namespace silkern
