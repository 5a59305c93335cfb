// Launch of the cache's attention: how many columns a CTA takes and how many
// CTAs share a work item's keys.
#include <atomic>
#include <numeric>

#include "attend_plan.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "silkern_b200.h"

namespace silkern {

namespace {

// About two seconds.
std::atomic<int64_t> wait_bound{4000000000};

}  // namespace

int64_t attend_wait_bound() { return wait_bound.load(std::memory_order_relaxed); }

int multiprocessors() {
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return 148;
  }
  return n;
}

namespace {

// One tensor's rows of a token and head: the pitch that divides its strides,
// and the strides in units of it. False where a row's number passes 31 bits.
struct Rows {
  int64_t pitch;
  uint32_t block, token, head;
};
bool find_rows(const PagedCache& c, int64_t block, int64_t token, int64_t head, Rows* r) {
  int64_t pitch = 0;
  if (c.num_blocks > 1) pitch = std::gcd(pitch, block);
  if (c.block.divisor > 1) pitch = std::gcd(pitch, token);
  if (c.kv_heads > 1) pitch = std::gcd(pitch, head);
  if (pitch == 0) pitch = 16;
  const int64_t last = (c.num_blocks - int64_t{1}) * (block / pitch) + (c.block.divisor - int64_t{1}) * (token / pitch) +
                       (c.kv_heads - int64_t{1}) * (head / pitch);
  if (last >= 0x7ffffffe) return false;
  *r = Rows{pitch, static_cast<uint32_t>(block / pitch), static_cast<uint32_t>(token / pitch),
            static_cast<uint32_t>(head / pitch)};
  return true;
}

}  // namespace

int set_rows(PagedCache& c) {
  Rows k, v;
  if (!find_rows(c, c.k_block, c.k_token, c.k_head, &k) ||
      !find_rows(c, c.v_block, c.v_token, c.v_head, &v)) {
    return SILKERN_E_CACHE;
  }
  c.k_block_rows = k.block;
  c.k_token_rows = k.token;
  c.k_head_rows = k.head;
  c.k_pitch = k.pitch;
  c.v_block_rows = v.block;
  c.v_token_rows = v.token;
  c.v_head_rows = v.head;
  c.v_pitch = v.pitch;
  return SILKERN_OK;
}

int launch_attend(AttendArgs& a, int key_dim, int type, cudaStream_t stream) {
  a.wait_cycles = attend_wait_bound();
  const bool latent = key_dim == 576, half = type == SILKERN_F16;
  const int32_t group = a.heads_per_kv;
  // Queries that may share a CTA's keys: one for a selected row; for
  // sequences as many as they have on average.
  const int64_t together = a.slots != nullptr ? 1 : (static_cast<int64_t>(a.rows) + a.sequences - 1) / a.sequences;
  const int64_t want = together * group;
  // A latent cache's fp16 queries have three parts: 64 columns of them do not
  // fit the shared memory beside the keys.
  const int widest = latent && half ? 32 : 64;
  int columns = want <= 16 ? 16 : want <= 32 || widest == 32 || (latent && group <= 32) ? 32 : 64;
  const int64_t sms = multiprocessors();
  int32_t per;
  int64_t blocks, items, live, tiles;
  while (true) {
    per = a.slots != nullptr || group >= columns ? 1 : columns / group;
    blocks = (group + columns - 1) / columns;
    items = a.slots != nullptr ? a.rows : (a.rows + static_cast<int64_t>(per - 1) * a.sequences) / per;
    int64_t busy = a.slots != nullptr ? a.rows : (a.rows + per - 1) / per;
    if (a.slots == nullptr && busy < a.sequences) busy = a.sequences < a.rows ? a.sequences : a.rows;
    live = busy * a.cache.kv_heads * blocks;
    int64_t keys = a.slots != nullptr ? a.width : static_cast<int64_t>(a.table_width) * a.cache.block.divisor;
    if (a.slots == nullptr && a.window != 0) {
      // This rank's share of what a CTA's queries see, and a run of owned tokens more.
      const int64_t seen = (static_cast<int64_t>(a.window) + a.sinks + per) / a.own.group.divisor * a.own.interleave.divisor +
                           2 * a.own.interleave.divisor;
      if (seen < keys) keys = seen;
    }
    tiles = (keys + 127) / 128;
    // While clusters over all keys still leave half of the SMs without work,
    // half the columns to a CTA: its queries are split, and its outputs
    // joined, in half the time (one row of 128 heads: 21.4 -> 12.5 us).
    if (columns == 16 || live * 2 * (tiles < 8 ? tiles : 8) > sms) break;
    columns /= 2;
  }
  const int64_t units = items * a.cache.kv_heads * blocks, pipes = !latent && columns <= 32 ? 2 : 1;
  if (units > 0x3fffffff) return SILKERN_E_SHAPE;
  AttendPlan plan;
  plan.per = make_fastdiv(static_cast<uint32_t>(per));
  plan.group = make_fastdiv(static_cast<uint32_t>(group));
  plan.blocks = static_cast<int32_t>(blocks);
  plan.units = static_cast<uint32_t>(units);
  // Few work items: CTAs share each item's keys, as a cluster of up to 16 that
  // leaves room for a cluster of every item, and of the sizes that give a
  // pipeline equally many tiles at most the smallest. Clusters come in any
  // size, since SMs do: of a B200's 148, clusters of 8 reach 120, of 9 or 3
  // 135, of 6 132.
  unsigned cluster = 1;
  if (live * 2 <= sms) {
    int64_t least = (tiles + pipes - 1) / pipes;  // tiles of a pipeline
    for (unsigned size = 2; size <= kMostCluster; ++size) {
      const int64_t ranks = size * pipes, most = (tiles + ranks - 1) / ranks;
      if (most < least && tiles >= ranks && units * size <= 0x7fffffff && live <= resident_clusters(size)) {
        cluster = size;
        least = most;
      }
    }
  }
  int64_t grid;
  if (cluster > 1 || (pipes > 1 && units <= sms && tiles >= pipes)) {
    plan.whole = 0;
    grid = units * cluster;
  } else {
    // Whole rounds of an item to each pipeline. What is left over after them is
    // split: over the pipelines of a CTA where these do not fill half a round,
    // over those of two CTAs where they do not fill a quarter (with one
    // pipeline, half). 512 equal items on 148 pipelines: 3.5 rounds, not 4.
    grid = (units + pipes - 1) / pipes < sms ? (units + pipes - 1) / pipes : sms;
    const int64_t round = grid * pipes, left = units % round;
    if (units > round && left > 0 && left <= grid / 2 && grid % 2 == 0) {
      cluster = 2;
      plan.whole = static_cast<uint32_t>(units - left);
    } else {
      plan.whole = static_cast<uint32_t>(pipes > 1 && left <= grid ? units - left : units);
    }
  }
  const int rc = set_rows(a.cache);
  if (rc != SILKERN_OK) return rc;
  AttendLaunch l{columns, half, static_cast<unsigned>(grid), cluster, stream};
  return key_dim == 64 ? launch_dim64(a, plan, l) : key_dim == 128 ? launch_dim128(a, plan, l) : launch_latent(a, plan, l);
}

}  // namespace silkern

extern "C" int64_t silkern_attend_wait_bound_v1(int64_t cycles) {
  if (cycles < 0 || cycles > (int64_t{1} << 32)) return silkern::wait_bound.load(std::memory_order_relaxed);
  return silkern::wait_bound.exchange(cycles, std::memory_order_relaxed);
}
