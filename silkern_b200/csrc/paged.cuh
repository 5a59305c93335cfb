// The 8-bit paged cache as the kernels see it, and which of its tokens one
// query sees.
//
// A page ("block") holds block_size consecutive rank-local tokens; every
// (page, head) pair has one float32 scale for its keys and one for its
// values, so the stored value is scale * e4m3 code. With key_dim 576 the
// cache is latent: one tensor, whose first 512 columns are the values too.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "fastdiv.cuh"

namespace silkern {

constexpr uint32_t kAllLanes = 0xffffffffu;

// A load that stays behind griddepcontrol.wait, and takes the coherent path:
// the grid before may have written what it reads.
__device__ __forceinline__ int32_t load_int(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

struct PagedCache {
  const uint8_t* k;
  const uint8_t* v;  // the keys again for a latent cache
  const float* k_scale;  // (num_blocks, kv_heads)
  const float* v_scale;
  int64_t k_block, k_token, k_head;  // strides in bytes, multiples of 16
  int64_t v_block, v_token, v_head;
  // The same in rows of a common pitch, which divides the strides (attention only).
  uint32_t k_block_rows, k_token_rows, k_head_rows, v_block_rows, v_token_rows, v_head_rows;
  int64_t k_pitch, v_pitch;
  uint32_t num_blocks;
  uint32_t kv_heads;
  FastDiv block;  // by block_size
};

// Context-parallel ownership: token t is rank (t / interleave) % dcp's.
struct Ownership {
  FastDiv group;       // by dcp_size * interleave
  FastDiv interleave;
  uint32_t rank_first; // dcp_rank * interleave

  // How many of the positions [0, x) this rank holds.
  __device__ __forceinline__ uint32_t owned_before(uint32_t x) const {
    const uint32_t q = fastdiv(x, group);
    const uint32_t r = x - q * group.divisor;
    const uint32_t mine = r > rank_first ? r - rank_first : 0u;
    return q * interleave.divisor + (mine < interleave.divisor ? mine : interleave.divisor);
  }
  // The position of rank-local token l.
  __device__ __forceinline__ uint32_t position(uint32_t l) const {
    const uint32_t q = fastdiv(l, interleave);
    return q * group.divisor + rank_first + (l - q * interleave.divisor);
  }
};

struct AttendArgs {
  PagedCache cache;
  const void* q;  // (rows, heads, key_dim), strides in elements
  int64_t q_row, q_head;
  void* out;  // (rows, heads, value_dim)
  int64_t out_row, out_head;
  bool out_wide;  // rows of out start on 16-byte boundaries
  float* lse;  // (rows, heads), contiguous
  int32_t* status;
  int64_t wait_cycles;  // bound on a wait inside the kernel
  float scale_log2;  // softmax_scale * log2(e)
  int32_t rows, heads;
  int32_t heads_per_kv;
  // Selected rows: slots (rows, width), counts optional.
  const int32_t* slots;
  const int32_t* counts;
  int64_t slots_row;
  int32_t width;
  uint32_t total_slots;
  // Sequences: cu_tokens (sequences + 1), lengths, req_ids (sequences,).
  const int32_t* cu_tokens;
  const int32_t* lengths;
  const int32_t* req_ids;
  const int32_t* table;
  int64_t table_rows;
  uint32_t table_width;
  int32_t sequences;
  uint32_t window;  // 0: the whole context
  uint32_t sinks;
  Ownership own;
};

__device__ __forceinline__ void flag_status(int32_t* status, int32_t bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// Queries [first, first + count) of one sequence that attend together.
struct QuerySpan {
  int32_t row;       // row of q of the first query
  int32_t count;     // 0: nothing to do
  int32_t seq;
  int32_t position;  // position of the first query; below 0: it sees nothing
};

// The span of up to `per` queries that work item `item` stands for. Sequence
// b owns the items from (cu[b] + (per - 1) b) / per on, which leaves each
// sequence at least one for each `per` of its tokens, so that
// (rows + (per - 1) sequences) / per items cover any cu_tokens that ascends to
// at most `rows`, and one for each sequence where each has one token. The
// warp's lanes search together, 32 boundaries a step.
__device__ __forceinline__ int32_t first_item(const FastDiv& per, int32_t cu, int32_t b) {
  return static_cast<int32_t>(fastdiv(static_cast<uint32_t>(cu) + (per.divisor - 1) * static_cast<uint32_t>(b), per));
}
__device__ __forceinline__ QuerySpan find_span(const AttendArgs& a, int32_t item, const FastDiv& per) {
  const int32_t lane = threadIdx.x & 31;
  int32_t low = 0, high = a.sequences;  // the last b in [low, high) with first_item(b) <= item
  while (high - low > 1) {
    const int32_t step = (high - low + 31) / 32;
    const int32_t b = low + lane * step;
    bool before = false;
    if (b < high) {
      const int32_t cu = min(max(load_int(a.cu_tokens + b), 0), a.rows);
      before = first_item(per, cu, b) <= item;
    }
    const uint32_t hits = __ballot_sync(kAllLanes, before);
    const int32_t last = hits == 0 ? 0 : 31 - __clz(hits);
    low += last * step;
    high = min(high, low + step);
  }
  QuerySpan s{0, 0, low, 0};
  const int32_t begin = min(max(load_int(a.cu_tokens + low), 0), a.rows);
  const int32_t end = min(max(load_int(a.cu_tokens + low + 1), begin), a.rows);
  const int32_t chunk = item - first_item(per, begin, low);
  const int64_t row = begin + static_cast<int64_t>(chunk) * per.divisor;
  if (chunk < 0 || row >= end) return s;
  s.row = static_cast<int32_t>(row);
  s.count = min(static_cast<int32_t>(per.divisor), end - s.row);
  const int64_t position = static_cast<int64_t>(load_int(a.lengths + low)) - (end - s.row);
  s.position = static_cast<int32_t>(max(position, int64_t{-0x7fffffff}));
  if (load_int(a.lengths + low) < end - begin && lane == 0) flag_status(a.status, 2);
  return s;
}

// Key numbers are 32-bit integers, and so are those a few tiles past the last.
constexpr uint32_t kMostKeys = 0x7fffffffu - 4096u;

// The keys that one work item reads, in order: j in [0, n).
struct KeyList {
  const int32_t* source;  // the row's slots, or the request's table row
  int32_t n;
  int32_t table;          // whether `source` is a table row
  uint32_t sinks_end;     // rank-local sink tokens [0, sinks_end) come first,
  uint32_t skip;          // then local token j + skip
  uint32_t table_width;
};

struct Key {
  uint32_t block, offset;
  int32_t position;  // global position (0 for a selected slot)
  bool valid;
};

__device__ __forceinline__ KeyList selected_keys(const AttendArgs& a, int32_t row) {
  KeyList l{a.slots + row * a.slots_row, a.width, 0, 0, 0, 0};
  if (a.counts != nullptr) {
    const int32_t c = load_int(a.counts + row);
    l.n = min(max(c, 0), a.width);
    if (c != l.n && (threadIdx.x & 31) == 0) flag_status(a.status, 2);
  }
  return l;
}

// The keys that any query of the span sees: the sinks and the union of the
// windows, clipped to this rank's tokens.
__device__ __forceinline__ KeyList window_keys(const AttendArgs& a, const QuerySpan& s) {
  KeyList l{nullptr, 0, 1, 0, 0, a.table_width};
  const int32_t req = load_int(a.req_ids + s.seq);
  if (req < 0 || req >= a.table_rows) {
    if ((threadIdx.x & 31) == 0) flag_status(a.status, 1);
    return l;
  }
  l.source = a.table + static_cast<int64_t>(req) * a.table_width;
  const int64_t last = static_cast<int64_t>(s.position) + s.count;  // positions below this are seen
  if (last <= 0) return l;
  const uint32_t end = static_cast<uint32_t>(last);
  const int64_t from = a.window == 0 ? 0 : static_cast<int64_t>(s.position) + 1 - a.window;
  const uint32_t begin = from > 0 ? static_cast<uint32_t>(from) : 0u;
  const uint32_t tail_end = a.own.owned_before(end);
  const uint32_t tail_begin = a.own.owned_before(begin);
  const uint32_t head_end = a.window == 0 ? 0u : a.own.owned_before(min(a.sinks, begin));
  l.sinks_end = head_end;
  l.skip = tail_begin - head_end;
  const uint32_t n = head_end + (tail_end - tail_begin);
  l.n = static_cast<int32_t>(min(n, kMostKeys));
  if (n > kMostKeys && (threadIdx.x & 31) == 0) flag_status(a.status, 2);
  return l;
}

// fetch: the one dependent load of key j (a slot or a table entry), issued
// ahead, for lists that are not empty; locate: what that value says. The load
// is unconditional, at a place inside the list, so that nothing waits for it
// before locate.
__device__ __forceinline__ uint32_t local_token(const KeyList& l, uint32_t j) {
  return j < l.sinks_end ? j : j + l.skip;
}
__device__ __forceinline__ int32_t fetch_key(const AttendArgs& a, const KeyList& l, int32_t j) {
  uint32_t at = min(j, l.n - 1);
  if (l.table) at = min(fastdiv(local_token(l, at), a.cache.block), l.table_width - 1);
  return load_int(l.source + at);
}
__device__ __forceinline__ Key locate_key(const AttendArgs& a, const KeyList& l, int32_t j, int32_t fetched) {
  Key k{0u, 0u, 0, false};
  if (!l.table) {
    k.valid = j < l.n && static_cast<uint32_t>(fetched) < a.total_slots;  // negative ones are above
    if (k.valid) {
      k.block = fastdiv(fetched, a.cache.block);
      k.offset = fetched - k.block * a.cache.block.divisor;
    }
    return k;
  }
  const uint32_t local = local_token(l, j), page = fastdiv(local, a.cache.block);
  k.valid = j < l.n && page < l.table_width && static_cast<uint32_t>(fetched) < a.cache.num_blocks;
  if (k.valid) {
    k.block = fetched;
    k.offset = local - page * a.cache.block.divisor;
    k.position = static_cast<int32_t>(a.own.position(local));
  }
  return k;
}
// Whether an unusable value deserves SILKERN_STATUS_BAD_SLOT: a slot past the
// cache, or a visible token whose page is not in the table row or the cache.
// (-1 in a selection row is padding.)
__device__ __forceinline__ bool bad_key(const KeyList& l, int32_t j, int32_t fetched, const Key& k) {
  return j < l.n && !k.valid && (l.table || fetched >= 0);
}

}  // namespace silkern
