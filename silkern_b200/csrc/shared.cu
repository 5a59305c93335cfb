// Attention of sequences in groups that share their first tokens: the plan, the
// joining of what the GPU's SMs found, and the entry points.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "attend_plan.cuh"
#include "cache_checks.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "shared_plan.cuh"
#include "silkern_b200.h"

namespace silkern {

namespace {

// ---------------------------------------------------------------- the plan

constexpr int kPlanThreads = 1024;

// A segment's tokens, keys and table row.
struct Segment {
  int32_t seq, seqs;
  int32_t token, tokens;
  int32_t key_first, key_end;  // rank-local
  int32_t table_row;
  int32_t length;  // of a sequence
};

// Groups' first sequences, prefixes, the longest length of each, and their first
// items, in shared memory as far as there is room; else where the call has them,
// and in the workspace.
constexpr int kHeldGroups = 1024;
struct Groups {
  int32_t cut[kHeldGroups + 1], prefix[kHeldGroups], longest[kHeldGroups], first[kHeldGroups];
};
__device__ __forceinline__ int32_t cut_of(const SharedArgs& a, const Groups& m, int32_t g) {
  return a.groups <= kHeldGroups ? m.cut[g] : a.cut(g);
}
__device__ __forceinline__ int32_t prefix_of(const SharedArgs& a, const Groups& m, int32_t g) {
  return a.groups <= kHeldGroups ? m.prefix[g] : load_int(a.prefixes + g);
}
__device__ __forceinline__ int32_t group_of(const SharedArgs& a, const Groups& m, int32_t seq) {  // -1: none
  if (seq < cut_of(a, m, 0) || seq >= cut_of(a, m, a.groups)) return -1;
  return last_at_most(a.groups, seq, [&](int32_t i) { return cut_of(a, m, i); });
}

// What a thread loads for its segment, before the groups are known.
struct Known {
  int32_t token, end, length, table_row;
};
__device__ __forceinline__ Known know_sequence(const SharedArgs& a, int32_t seq) {
  return {a.cu(seq), a.cu(seq + 1), load_int(a.lengths + seq), load_int(a.req_ids + seq)};
}

__device__ __forceinline__ Segment find_segment(const SharedArgs& a, const Groups& m, int32_t index, const Known& known) {
  Segment s{};
  s.token = known.token;
  s.tokens = max(known.end - known.token, 0);
  s.table_row = known.table_row;
  if (index < a.groups) {
    s.seq = cut_of(a, m, index);
    s.seqs = cut_of(a, m, index + 1) - s.seq;
    const int32_t longest = a.groups <= kHeldGroups ? m.longest[index] : a.limits()[index];
    s.key_end = a.keys_below(min(longest, prefix_of(a, m, index)));
  } else {
    s.seq = index - a.groups;
    s.seqs = 1;
    s.length = known.length;
    if (s.tokens > 0 && s.length < s.tokens) flag_status(a.status, SILKERN_STATUS_BAD_LENGTH);
    s.key_end = a.keys_below(s.length);
    const int32_t group = group_of(a, m, s.seq);
    if (group >= 0) s.key_first = a.keys_below(prefix_of(a, m, group));
  }
  if (s.tokens > 0 && s.key_end > s.key_first && (s.table_row < 0 || s.table_row >= a.table_rows)) {
    flag_status(a.status, SILKERN_STATUS_BAD_REQUEST);
    s.tokens = 0;
  }
  return s;
}

// Rows [256 block, ...) of a segment: how many, and the keys that they see.
__device__ __forceinline__ SharedItem item_of(const SharedArgs& a, const Segment& s, bool prefix, int32_t block) {
  SharedItem it{};
  it.row = block * kBlockRows;
  it.rows = min(s.tokens * a.heads_per_kv - it.row, kBlockRows);
  it.key_begin = s.key_first & ~15;
  it.key_first = s.key_first;
  it.key_end = s.key_end;
  if (!prefix && s.tokens > 1) {  // up to its last query's
    const int32_t last = static_cast<int32_t>(fastdiv(it.row + it.rows - 1, a.per_kv));
    const int64_t position = static_cast<int64_t>(s.length) - (s.tokens - last);
    it.key_end = position < 0 ? 0 : min(it.key_end, a.keys_below(static_cast<int32_t>(position + 1)));
  }
  it.tiles = it.key_end > it.key_first
                 ? static_cast<int32_t>((static_cast<int64_t>(it.key_end) - it.key_begin + kSharedTile - 1) / kSharedTile)
                 : 0;
  it.table_row = s.table_row;
  it.token = s.token;
  it.seq = s.seq;
  it.seqs = s.seqs;
  it.prefix = prefix ? 1 : 0;
  return it;
}

// One CTA lays out the items: a thread for each segment, and prefix sums over
// them. Fewer dependent loads than launches cost: 4.7 us alone in a graph for 4
// sequences, 6.2 for 256 in 5 groups. A thread goes through its segment's blocks of
// 256 rows one by one, which no decode step notices: prompts do, by 0.13 us for each
// block of the longest segment (4 times 2048 queries of 8 heads behind a prefix,
// 256 blocks: 43 us by itself and cold, where 4 sequences take 9, of a call of 3.5 ms).
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const __grid_constant__ SharedArgs a, int32_t ctas) {
  __shared__ int64_t sums[3][32];
  __shared__ Groups groups;
  pdl_wait();
  pdl_launch_dependents();
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t segments = a.groups + a.sequences;
  const bool held = a.groups <= kHeldGroups;
  // All loads that wait for none, and whether sequences or groups descend: such a
  // call could have more items than the workspace holds, and has none.
  const int32_t my_seq = static_cast<int32_t>(threadIdx.x) - a.groups;
  Known known{};
  if (my_seq >= 0 && my_seq < a.sequences) known = know_sequence(a, my_seq);
  bool descends = known.end < known.token;
  for (int32_t i = kPlanThreads - a.groups + static_cast<int32_t>(threadIdx.x); i < a.sequences; i += kPlanThreads) {
    descends = descends || (i >= 0 && a.cu(i + 1) < a.cu(i));
  }
  for (int32_t g = threadIdx.x; g < a.groups; g += kPlanThreads) {
    const int32_t first = a.cut(g), last = a.cut(g + 1);
    descends = descends || last < first;
    if (held) {
      groups.cut[g] = first;
      if (g + 1 == a.groups) groups.cut[g + 1] = last;
      groups.prefix[g] = load_int(a.prefixes + g);
      groups.longest[g] = 0;
    }
  }
  descends = __syncthreads_or(descends);
  if (descends && threadIdx.x == 0) flag_status(a.status, SILKERN_STATUS_BAD_LENGTH);
  // Prefixes end where the last query of the group sees no further.
  if (descends) {
  } else if (held) {
    const int32_t index = threadIdx.x;
    if (index < a.groups) {
      const int32_t first = groups.cut[index], last = groups.cut[index + 1];
      if (last > first) known = {a.cu(first), a.cu(last), 0, load_int(a.req_ids + first)};
    }
    for (int32_t base = 0; base < segments; base += kPlanThreads) {
      const int32_t seq = base + index - a.groups;
      if (seq < 0 || seq >= a.sequences) continue;
      const Known k = base == 0 ? known : know_sequence(a, seq);
      const int32_t group = k.end > k.token ? group_of(a, groups, seq) : -1;
      if (group >= 0) atomicMax(&groups.longest[group], k.length);
    }
  } else {
    for (int32_t g = warp; g < a.groups; g += kPlanThreads / 32) {
      const int32_t first = a.cut(g), last = a.cut(g + 1);
      int32_t most = 0;
      for (int32_t s = first + lane; s < last; s += 32) {
        if (a.cu(s + 1) > a.cu(s)) most = max(most, load_int(a.lengths + s));
      }
      most = __reduce_max_sync(kAllLanes, most);
      if (lane == 0) a.limits()[g] = most;
    }
  }
  __syncthreads();
  int64_t before[3] = {0, 0, 0};  // items, units, rows of second copies
  for (int32_t base = 0; base < segments; base += kPlanThreads) {
    const int32_t index = base + threadIdx.x;
    Segment s{};
    int32_t blocks = 0;
    const bool prefix = index < a.groups;
    int64_t mine[3] = {0, 0, 0};
    if (index < segments && !descends) {
      if (base > 0 || !held) {
        if (index >= a.groups) {
          known = know_sequence(a, index - a.groups);
        } else {
          const int32_t first = a.cut(index), last = a.cut(index + 1);
          known = Known{};
          if (last > first) known = {a.cu(first), a.cu(last), 0, load_int(a.req_ids + first)};
        }
      }
      s = find_segment(a, groups, index, known);
      if (s.tokens > 0 && s.key_end > s.key_first) {
        blocks = (s.tokens * a.heads_per_kv + kBlockRows - 1) / kBlockRows;
        mine[0] = blocks;
        for (int32_t b = 0; b < blocks; ++b) {
          // (A prefix's blocks are alike, but for the last's rows.)
          if (prefix && b == 1) {
            mine[1] *= blocks - 1;
            b = blocks - 1;
          }
          const SharedItem it = item_of(a, s, prefix, b);
          mine[1] += units_of(it.tiles, it.rows);
          if (it.rows <= kSlotRows) mine[2] += it.rows;
        }
      }
    }
    int64_t upto[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int64_t x = mine[k];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(kAllLanes, x, d);
        if (lane >= d) x += y;
      }
      upto[k] = x;
      if (lane == 31) sums[k][warp] = x;
    }
    __syncthreads();
    int64_t all[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int64_t x = sums[k][lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(kAllLanes, x, d);
        if (lane >= d) x += y;
      }
      all[k] = __shfl_sync(kAllLanes, x, 31);
      const int64_t warps_before = __shfl_sync(kAllLanes, x, max(warp - 1, 0));
      upto[k] += before[k] - mine[k] + (warp > 0 ? warps_before : 0);
    }
    const int32_t first_item = blocks > 0 ? static_cast<int32_t>(upto[0]) : -1;
    if (prefix) {
      a.first()[index] = first_item;
      if (held) groups.first[index] = first_item;
    }
    for (int32_t b = 0; b < blocks; ++b) {
      SharedItem it = item_of(a, s, prefix, b);
      it.begin = upto[1];
      it.extra = static_cast<int32_t>(upto[2]);
      upto[1] += units_of(it.tiles, it.rows);
      if (it.rows <= kSlotRows) upto[2] += it.rows;
      *a.item(static_cast<int32_t>(upto[0]) + b) = it;
    }
    __syncthreads();
    if (index >= a.groups && index < segments) {  // what joining has to know
      const int32_t seq = index - a.groups, group = descends ? -1 : group_of(a, groups, seq);
      int4 record = make_int4(first_item, known.token, -1, known.token);
      if (group >= 0) {
        record.z = held ? groups.first[group] : a.first()[group];
        record.w = a.cu(cut_of(a, groups, group));
      }
      a.records()[seq] = record;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) before[k] += all[k];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    SharedHeader h;
    h.units = before[1] * a.cache.kv_heads;
    h.share = max((h.units + ctas - 1) / ctas, static_cast<int64_t>(kLeastUnits));
    h.items = static_cast<int32_t>(before[0]);
    h.failed = 0;
    *a.header() = h;
  }
}

// ---------------------------------------------------------------- joining

// The fragments of one row of an item: the first CTA's, and those of the CTAs
// that went on with it.
struct Parts {
  int64_t first, copy, next;  // partial rows; copy -1: none
  int32_t count;              // of fragments
  int32_t both;               // 1: the two slots have a copy each
};

// `first`: the segment's first item, `row` the row's number in the segment.
__device__ __forceinline__ Parts find_parts(const SharedArgs& a, int32_t first, int32_t row, int32_t kv, int64_t share, int64_t place) {
  row = max(row, 0);  // (below it in a call whose groups descend)
  const SharedItem* it = a.item(max(first, 0) + row / kBlockRows);
  // (Loads that wait for one another cost more than some too many.)
  const int32_t tiles = load_int(&it->tiles), rows = load_int(&it->rows), extra = load_int(&it->extra);
  const int64_t begin = __ldcg(&it->begin);
  const int32_t r = row % kBlockRows;
  const int64_t zero = begin * a.cache.kv_heads + kv * units_of(tiles, rows) + units_of_start(rows);
  const int64_t c0 = zero / share, c1 = (zero + static_cast<int64_t>(tiles - 1) * units_of_tile(rows)) / share;
  Parts p{place, -1, a.at.starts + (c0 + 1) * kBlockRows + r, static_cast<int32_t>(c1 - c0 + 1), 0};
  if (rows <= kSlotRows) {
    p.both = 1;
    p.copy = a.at.copies + static_cast<int64_t>(extra) * a.cache.kv_heads + static_cast<int64_t>(kv) * rows + r;
  }
  if (first < 0 || tiles <= 0) p.count = 0;
  return p;
}
__device__ __forceinline__ int64_t part_at(const Parts& p, int32_t i) {
  const int32_t c = p.both ? i >> 1 : i;
  const bool second = p.both && (i & 1);
  if (c == 0) return second ? p.copy : p.first;
  return p.next + (c - 1) * int64_t{kBlockRows} + (second ? kSlotRows : 0);
}

__device__ __forceinline__ Parts parts_of_lane(const Parts& p, int32_t lane) {
  return {__shfl_sync(kAllLanes, p.first, lane), __shfl_sync(kAllLanes, p.copy, lane), __shfl_sync(kAllLanes, p.next, lane),
          __shfl_sync(kAllLanes, p.count, lane), __shfl_sync(kAllLanes, p.both, lane)};
}

// WARPS warps to a (query, head): one where there are many of them, eight where
// few rows have many fragments (a call with 64 of 37: 104 us for 113; with 512, 119
// for 125; with 1024, 139.3 for 138.4). A lane looks the group's
// fragments up, its neighbour the sequence's own; lanes weigh the fragments, then
// each warp adds up its share of them in order, and the first the warps'. Bound by
// the chain of loads: several heads to a warp were slower.
template <typename T, int DIM, int WARPS>
__global__ void __launch_bounds__(256) shared_join_kernel(const __grid_constant__ SharedArgs a) {
  constexpr int kEach = DIM / 32;  // columns of a lane
  __shared__ float partial[WARPS == 1 ? 1 : 8][DIM];
  pdl_wait();
  pdl_launch_dependents();
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t w = WARPS == 1 ? 0 : warp;
  const int64_t pair = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  const int64_t pairs = static_cast<int64_t>(a.rows) * a.heads;
  if (pair >= pairs) return;
  const int32_t token = static_cast<int32_t>(pair / a.heads), head = static_cast<int32_t>(pair - static_cast<int64_t>(token) * a.heads);
  if (token < a.cu(0) || token >= a.cu(a.sequences)) return;
  const int64_t share = __ldcg(&a.header()->share);
  const int32_t failed = load_int(&a.header()->failed);
  const int32_t seq = warp_last_at_most(a.sequences, token, [&](int32_t i) { return a.cu(i); });
  const int4 record = __ldcg(a.records() + seq);  // the sequence's first item and token, its group's
  const int32_t kv = static_cast<int32_t>(fastdiv(head, a.per_kv)), in_kv = head - kv * a.heads_per_kv;
  const bool own = lane & 1;
  const Parts mine = find_parts(a, own ? record.x : record.z, (token - (own ? record.y : record.w)) * a.heads_per_kv + in_kv, kv, share,
                                own ? pairs + pair : pair);
  const Parts part[2] = {parts_of_lane(mine, 0), parts_of_lane(mine, 1)};
  const int32_t n0 = part[0].count << part[0].both, n = n0 + (part[1].count << part[1].both);
  auto place = [&](int32_t i) { return i < n0 ? part_at(part[0], i) : part_at(part[1], i - n0); };
  // This lane's of the first 32 fragments.
  const int64_t first_at = lane < n ? place(lane) : 0;
  const float first_lse = lane < n ? __ldcg(a.part_lse() + first_at) : -INFINITY;
  float top = first_lse;
  for (int32_t i = lane + 32; i < n; i += 32) {
    const float l = __ldcg(a.part_lse() + place(i));
    top = l != l ? l : top != top ? top : fmaxf(top, l);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float l = __shfl_xor_sync(kAllLanes, top, d);
    top = l != l ? l : top != top ? top : fmaxf(top, l);
  }
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f, y[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) y[e] = 0.f;
  // Each round of 32 fragments: a lane has one's place and weight, and the
  // warps take turns with them, four on their way at once.
  for (int32_t i0 = 0; i0 < n; i0 += 32) {
    const int64_t at = i0 == 0 ? first_at : i0 + lane < n ? place(i0 + lane) : 0;
    const float weight = i0 + lane >= n ? 0.f : exp2f((i0 == 0 ? first_lse : __ldcg(a.part_lse() + at)) - base);
    float sum = weight;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
    total += sum;
    const int32_t left = min(32, n - i0);
    for (int32_t j0 = w; j0 < left; j0 += 4 * WARPS) {
      float x[4][kEach], by[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int32_t j = j0 + k * WARPS;
        by[k] = __shfl_sync(kAllLanes, weight, j & 31);
        const int64_t from = __shfl_sync(kAllLanes, at, j & 31);
        if (j >= left) by[k] = 0.f;
#pragma unroll
        for (int e = 0; e < kEach; ++e) x[k][e] = 0.f;
        if (by[k] != 0.f) {  // a fragment without weight has no outputs
          const float* p = a.part_out() + from * DIM + lane * kEach;
          if constexpr (kEach == 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
            x[k][0] = v.x;
            x[k][1] = v.y;
            x[k][2] = v.z;
            x[k][3] = v.w;
          } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(p));
            x[k][0] = v.x;
            x[k][1] = v.y;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) y[e] = fmaf(by[k], x[k][e], y[e]);
      }
    }
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) partial[warp][lane * kEach + e] = y[e];
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      y[e] = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) y[e] += partial[i][lane * kEach + e];
    }
  }
  float inverse = total == 0.f ? 0.f : 1.f / total, lse = (top + log2f(total)) * 0.69314718055994531f;
  if (failed != 0) inverse = lse = NAN;
  T* out = static_cast<T*>(a.out) + token * a.out_row + head * a.out_head + lane * kEach;
  T rounded[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) rounded[e] = static_cast<T>(y[e] * inverse);
  if (a.out_wide) {
    if constexpr (kEach == 4) {
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(rounded);
    } else {
      *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(rounded);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e) out[e] = rounded[e];
  }
  if (lane == 0) a.lse[pair] = lse;
}

template <typename T, int DIM>
int launch_join(const SharedArgs& a, cudaStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(a.rows) * a.heads;
  if (pairs <= 4 * kMostCtas) return launch_pdl(shared_join_kernel<T, DIM, 8>, static_cast<unsigned>(pairs), 256, 0, 1, stream, a);
  return launch_pdl(shared_join_kernel<T, DIM, 1>, static_cast<unsigned>((pairs + 7) / 8), 256, 0, 1, stream, a);
}

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// The workspace's layout. Every (row, head) has a partial result of its group's
// prefix and one of its own tokens, whether it sees both or not.
int lay_out(int64_t rows, int32_t heads, int32_t kv_heads, int32_t dim, int64_t sequences, int64_t groups, SharedLayout* at) {
  if (rows < 1 || rows > 0x7fffffff || sequences < 1 || sequences > 0x3fffffff || groups < 1 || groups > 0x3fffffff) return SILKERN_E_SHAPE;
  if (sequences + groups > 0x7fffffff - kPlanThreads) return SILKERN_E_SHAPE;  // the plan's rounds end below 2^31
  if (heads < 1 || heads > 65535 || kv_heads < 1 || heads % kv_heads != 0) return SILKERN_E_HEADS;
  if (dim != 64 && dim != 128) return SILKERN_E_CACHE;
  if (rows * heads > 0x3fffffff) return SILKERN_E_SHAPE;
  const int64_t each = rows * (heads / kv_heads), segments = sequences + groups;
  at->limits = 64;
  at->first = at->limits + 4 * groups;
  at->records = round_up(at->first + 4 * groups, 64);
  at->items = round_up(at->records + 16 * sequences, 64);
  at->most_items = 2 * (each / kBlockRows) + segments;
  at->starts = 2 * rows * heads;
  at->copies = at->starts + int64_t{kMostCtas} * kBlockRows;
  const int64_t partial = at->copies + kv_heads * std::min(2 * each, kSlotRows * segments);
  at->lse = at->items + 64 * at->most_items;
  at->out = round_up(at->lse + 4 * partial, 64);
  at->bytes = at->out + 4 * partial * dim;
  return SILKERN_OK;
}

}  // namespace
}  // namespace silkern

using namespace silkern;

extern "C" int64_t silkern_shared_workspace_v1(int64_t rows, int32_t heads, int32_t kv_heads, int32_t dim, int64_t sequences,
                                               int64_t groups) {
  SharedLayout at{};
  const int rc = lay_out(rows, heads, kv_heads, dim, sequences, groups, &at);
  return rc == SILKERN_OK ? at.bytes : -rc;
}

extern "C" int silkern_attend_shared_v1(const silkern_cache_v1* cache, const void* q, int64_t q_row, int64_t q_head,
                                        int32_t type, int64_t rows, int32_t heads, const int32_t* cu_tokens,
                                        const int32_t* lengths, const int32_t* req_ids, int64_t sequences,
                                        const int32_t* cu_groups, const int32_t* prefixes, int64_t groups,
                                        const int32_t* block_table, int64_t table_rows, int64_t table_width,
                                        int32_t dcp_size, int32_t dcp_rank, int32_t dcp_interleave, void* out,
                                        int64_t out_row, int64_t out_head, float* lse, float softmax_scale,
                                        void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  SharedArgs a{};
  int rc = check_cache(cache, &a.cache);
  if (rc != SILKERN_OK) return rc;
  if (cache->key_dim == 576) return SILKERN_E_CACHE;
  if (!q || !out || !lse || !cu_tokens || !lengths || !req_ids || !cu_groups || !prefixes || !block_table || !workspace) {
    return SILKERN_E_NULL;
  }
  if (type != SILKERN_BF16 && type != SILKERN_F16) return SILKERN_E_TYPE;
  rc = lay_out(rows, heads, cache->kv_heads, cache->key_dim, sequences, groups, &a.at);
  if (rc != SILKERN_OK) return rc;
  if (table_rows < 1 || table_width < 1 || table_width > 0x7fffffff) return SILKERN_E_SHAPE;
  if (workspace_bytes < a.at.bytes) return SILKERN_E_SCRATCH;
  if (q_row % 8 != 0 || q_head % 8 != 0 || reinterpret_cast<uintptr_t>(q) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return SILKERN_E_CACHE;
  }
  a.scale_log2 = std::fabs(softmax_scale) * 1.4426950408889634f;
  a.q_sign = softmax_scale < 0.f ? -1.f : 1.f;
  if (!std::isfinite(a.scale_log2)) return SILKERN_E_ATTEND;
  rc = check_owner(cache->block_size, dcp_size, dcp_rank, dcp_interleave, &a.own);
  if (rc != SILKERN_OK) return rc;
  const Place written[3] = {Place(out, 2 * int64_t{cache->value_dim}).along(rows, 2 * out_row).along(heads, 2 * out_head),
                            Place(lse, 4 * rows * heads), Place(workspace, workspace_bytes)};
  const Place read[11] = {Place(q, 2 * int64_t{cache->key_dim}).along(rows, 2 * q_row).along(heads, 2 * q_head),
                          place_of_keys(cache), place_of_values(cache), place_of_scales(cache, cache->k_scale),
                          place_of_scales(cache, cache->v_scale), Place(cu_tokens, 4 * (sequences + 1)),
                          Place(lengths, 4 * sequences), Place(req_ids, 4 * sequences), Place(cu_groups, 4 * (groups + 1)),
                          Place(prefixes, 4 * groups), Place(block_table, 4 * table_rows * table_width)};
  if (shares(written, read)) return SILKERN_E_ALIAS;
  a.q = q;
  a.q_row = q_row;
  a.q_head = q_head;
  a.out = out;
  a.out_row = out_row;
  a.out_head = out_head;
  a.lse = lse;
  a.status = status;
  a.rows = static_cast<int32_t>(rows);
  a.heads = heads;
  a.heads_per_kv = heads / cache->kv_heads;
  a.per_kv = make_fastdiv(static_cast<uint32_t>(a.heads_per_kv));
  a.out_wide = out_row % 4 == 0 && out_head % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
  a.work = static_cast<uint8_t*>(workspace);
  a.wait_cycles = attend_wait_bound();
  a.runs = cache->block_size % 16 == 0;
  a.sequences = static_cast<int32_t>(sequences);
  a.groups = static_cast<int32_t>(groups);
  a.cu_tokens = cu_tokens;
  a.lengths = lengths;
  a.req_ids = req_ids;
  a.cu_groups = cu_groups;
  a.prefixes = prefixes;
  a.table = block_table;
  a.table_rows = table_rows;
  a.table_width = static_cast<uint32_t>(table_width);
  rc = set_rows(a.cache);
  if (rc != SILKERN_OK) return rc;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  const int sms = multiprocessors(), ctas = sms < kMostCtas ? sms : kMostCtas;
  rc = launch_pdl(shared_plan_kernel, 1, kPlanThreads, 0, 1, on, a, ctas);
  if (rc != SILKERN_OK) return rc;
  const bool half = type == SILKERN_F16, narrow = cache->key_dim == 64;
  rc = narrow ? launch_shared_dim64(a, half, ctas, on) : launch_shared_dim128(a, half, ctas, on);
  if (rc != SILKERN_OK) return rc;
  if (narrow) return half ? launch_join<__half, 64>(a, on) : launch_join<__nv_bfloat16, 64>(a, on);
  return half ? launch_join<__half, 128>(a, on) : launch_join<__nv_bfloat16, 128>(a, on);
}
