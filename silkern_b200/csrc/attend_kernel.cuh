// Attention over the 8-bit paged cache on the fifth-generation tensor core.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(softmax_scale q . k_j),  lse = log sum_j p_j
//
// The tensor core reads the cache's e4m3 codes as they lie in the cache: no
// element of K or V is converted. A CTA takes NH columns, (query, head) pairs
// that read one cache head, and walks that head's keys in tiles of 128:
//
//   S^T (128 keys x columns) = K (128 x dim) Q^T,      M = keys
//   O^T (dim x columns)     += V^T (dim x 128) P^T,    M = value dim
//
// K is the K-major A operand and V, stored the same way, the M-major one, so
// a latent cache's rows serve as both from one copy in shared memory. Q and P
// are split into T parts of 8 bits whose sum is the number: an e4m3 part holds
// 4 significant bits, a second holds what the first left, scaled or not, so
// that a bf16 query is exact in two parts and an fp16 one in three. The
// parts of P after the first are e5m2, for range: they end at 2^-17 instead of
// 2^-10, below a reference that follows each tile's largest weight, so that many small
// weights keep their sum beside a large one. Q's parts lie side by side along
// N (their scores are added in float32, each with its own scale); P's parts
// are added up in the accumulator.
//
// Weights: with s_j = log2(p_j), u_j = s_j + log2(vscale_j) and R a reference
// near the tile's largest u, P'_j = 2^(u_j - R + 5) goes to the tensor core, and
// 2^(s_j - Q) to the sum l: out = O 2^(R - Q) / (32 l), lse = (Q + log2 l) ln 2.
// R moves, and O is rescaled, only when a tile's largest u leaves [R - 4, R +
// 3.5]: e4m3 ends at 448 = 2^8.8. l, S and O are float32.
//
// The sum's own reference Q: as long as an item's value scales lie within
// 2^kUsual of 1, Q is R, and 2^(s_j - Q) is P'_j 2^-5 / vscale_j. R is at most
// the largest u so far, and at least 60 below it and 3.5 below the tile's, so
// that l is at most 2^31 keys of 2^(3.5 + kUsual + 60), in float32 with room;
// and P' of a key 40 below the largest s is above 2^(5 - 40 - 2 kUsual), which
// is not flushed. From the first tile with another scale on (0, whose values
// count nothing, goes into u as 2^-100) each warp keeps a Q of its own, the
// largest s of its keys, and takes a second exponential for the sum; at the
// item's end O and l come to one reference again. That holds for any scales in
// [2^-100, 2^100], in any order, and costs the usual ones 0 to 5 % (a flag of
// the tile, looked at behind the barrier that the maxima need anyway).
//
// A CTA is one or two pipelines, each a softmax of one key a thread and 16
// columns a warpgroup, warps that gather keys and values with cp.async (the TMA
// unit's four-row gathers took 61 cycles for 512 bytes of an SM here, these
// copies about 12), warps that split the queries, and one that issues the MMAs.
// The kernel takes all of an SM's shared memory, so a CTA stays on its SM and
// its pipelines walk through the work items; each role runs ahead as far as the
// buffers let it, and one item's start and end hide behind its neighbours'.
// Work items that are few, or left over after whole rounds, are split over
// their keys: by the pipelines of a CTA and of a thread-block cluster, which
// join their sums and outputs through (distributed) shared memory. No
// workspace, one launch.
//
// Measured: a decode step of 128 sequences, 8 heads of 128, window 4096 (1.02
// GB): 207 us, 4.9 TB/s, bound by memory. 256 rows of 512 latent keys, 128
// heads: 85 us, 428 TFLOP/s, bound by an item's start and end (four tiles
// between them). 4001 queries of a prompt, window 1024, heads of 64, fp16: 268
// us, bound by the softmax's instructions. One row over 131072 tokens: 81 us,
// 3.3 TB/s on the 80 SMs that clusters for 8 heads reach. With value scales
// outside 2^+-kUsual throughout: 5 (latent) to 37 % (prompt) longer.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "attend_plan.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "silkern_b200.h"
#include "tcgen05.cuh"

namespace silkern {

enum CacheShape { kDim64, kDim128, kLatent };

constexpr int kTile = 128;
// Value scales from 2^-kUsual to 2^kUsual share the sum's reference with the
// outputs': every page of values with a largest magnitude from 2^-15 to 2^32.
constexpr float kUsual = 24.f;
// All of an SM's shared memory that a CTA can have.
constexpr int kSharedMemory = 227 * 1024;

template <CacheShape SHAPE, int NH, int T>
struct Config {
  static constexpr bool kIsLatent = SHAPE == kLatent;
  static constexpr int kKeyDim = SHAPE == kDim64 ? 64 : SHAPE == kDim128 ? 128 : 576;
  static constexpr int kValueDim = SHAPE == kDim64 ? 64 : SHAPE == kDim128 ? 128 : 512;
  static constexpr int kWide = SHAPE == kDim64 ? 64 : 128;       // row bytes of the main chunks
  static constexpr int kMainKeys = kIsLatent ? 4 : 1;            // K chunks of kWide bytes
  static constexpr int kValues = kIsLatent ? 4 : 1;              // V chunks: M = 128 tiles of O^T
  static constexpr int kLoadChunks = kIsLatent ? 5 : 2;          // four wide ones and the tail; else keys, values
  static constexpr int kChunkBytes = kWide * kTile;
  static constexpr int kStageBytes = (kIsLatent ? 4 : 2) * kChunkBytes;
  static constexpr int kTailBytes = kIsLatent ? 64 * kTile : 0;  // a latent key's last 64 bytes
  // Pipelines: a narrow column block's softmax is a chain of short steps, and
  // two of them keep the memory busy.
  static constexpr int kPipes = !kIsLatent && NH <= 32 ? 2 : 1;
  static constexpr int kGroups = NH / 16;                        // softmax warpgroups, 16 columns each
  static constexpr int kSoftmax = kGroups * 128;
  static constexpr int kLoaders = kPipes == 2 || NH == 64 ? 2 : 4;  // gathering warps
  static constexpr int kSplitters = kPipes == 2 ? 1 : NH == 64 ? 5 : 3;  // query warps
  static constexpr int kPipeWarps = kGroups * 4 + kLoaders + kSplitters + 1;
  static_assert(kPipeWarps % 4 == 0, "a softmax warp's TMEM lanes go by its number in the CTA");
  static constexpr int kThreads = kPipes * kPipeWarps * 32;
  static constexpr int kQBytes = T * NH * kKeyDim;
  static constexpr int kPBytes = T * NH * kTile;
  // Columns of several queries see different keys. 64 columns of a latent
  // cache are one query's, so that its shared memory need not hold positions.
  static constexpr bool kSeveral = !(kIsLatent && NH == 64);
  static constexpr int kNoteBytes = kTile * ((kIsLatent ? 4 : 8) + (kSeveral ? 4 : 0)) + 16;  // a tile's scales, positions
  static constexpr int kMisc = NH * (12 + 4 + 8) + 320;
  // TMEM columns of a pipeline: outputs, and scores twice.
  static constexpr int kPipeColumns = kValues * NH + 2 * T * NH;
  static constexpr int kColumnsUsed = kPipes * kPipeColumns;
  static_assert(kColumnsUsed <= 512, "TMEM");
  static constexpr int kColumns = kColumnsUsed <= 128 ? 128 : kColumnsUsed <= 256 ? 256 : 512;
  static constexpr int kPipeBytes = kSharedMemory / kPipes / 1024 * 1024;
  static constexpr int kFixed = kQBytes + kPBytes + kMisc;
  static constexpr int kStageCost = kStageBytes + kNoteBytes + 16 * kLoadChunks;  // with its barriers
  static constexpr int kFit = (kPipeBytes - kFixed) / kStageCost;
  static constexpr int kStages = kIsLatent ? 2 : kFit < 8 ? kFit : 8;
  static constexpr int kTails = kIsLatent ? ((kPipeBytes - kFixed - 2 * kStageCost) >= 2 * kTailBytes ? 2 : 1) : 0;
  static_assert(kStages >= 2 && kFixed + kStages * kStageCost + kTails * kTailBytes <= kPipeBytes, "shared memory");
  // Ranks that may share an item, and the columns that their shares round up to.
  static constexpr int kMostRanks = kMostCluster * kPipes;
  // The chunk whose buffer is free again only after a tile's softmax, and
  // with it the tile's scales and positions.
  static constexpr int kNoteChunk = kIsLatent ? 0 : 1;
  // Offsets from the start of a pipeline's shared memory.
  static constexpr int kOffTail = kStages * kStageBytes;
  static constexpr int kOffQ = kOffTail + kTails * kTailBytes;
  static constexpr int kOffP = kOffQ + kQBytes;
  static constexpr int kOffMisc = kOffP + kPBytes;
  static_assert((NH + kMostRanks - 1) * kValueDim * 4 <= kOffP, "joining buffer");
};

// A work item as its query warps hand it to the softmax and the MMAs.
struct Handed {
  int32_t row, count, position;  // its queries
  int32_t kv, block;
  int32_t steps;                 // tiles; -1: no more items
  int32_t split;                 // whether its keys are split over ranks
};

// The small shared state of a pipeline, behind its tiles.
template <typename C, int NH>
struct __align__(16) Shared {
  int32_t best[3][NH];  // column maxima of a tile, as ordered integers
  alignas(16) float reference[NH];  // 5 - R of the columns' references R; read four at a time, like the factors
  alignas(16) float factor[2][NH];  // the columns' score factors, of this item and the next
  float k_scale[C::kStages][kTile];
  float v_scale[C::kIsLatent ? 1 : C::kStages][C::kIsLatent ? 1 : kTile];
  int32_t position[C::kSeveral ? C::kStages : 1][C::kSeveral ? kTile : 1];
  uint32_t valid[C::kStages][4];  // a bit for each key
  Handed handed[2];
  Handed last;          // the split item, as soon as it is known
  int32_t last_known;
  uint32_t unusual[C::kGroups];  // the last item with an unusual scale, counted from 1
  uint64_t full[C::kLoadChunks][C::kStages], empty[C::kLoadChunks][C::kStages];
  uint64_t scores[2], weights, done;
  uint64_t queries[2], queries_read, finished[2];
  uint64_t drained;
  uint32_t tmem;
  int32_t abort;
};

__device__ __forceinline__ int32_t ordered(float x) {
  const int32_t b = __float_as_int(x);
  return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float unordered(int32_t b) { return __int_as_float(b >= 0 ? b : b ^ 0x7fffffff); }

// A whole warp waits. A wait that ran out leaves *abort set, and every later
// wait returns after a try or two (some 4 us): the gathering and the MMAs end, a
// softmax runs through its item's tiles on whatever is there, so that its
// groups' barriers get the arrivals they count, and no further item begins.
__device__ __forceinline__ void warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int64_t bound) {
  mbar_wait(smem_addr(bar), parity, abort, bound);
  __syncwarp();
}

// Splits four numbers into T parts of one byte each. Parts of a query are
// e4m3, scaled by 16 from part to part. Of a weight's parts the first is e4m3
// and the others e5m2, all of one scale.
template <int T, bool WEIGHT>
__device__ __forceinline__ void split4(const float (&x)[4], uint32_t (&part)[T]) {
  float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const bool wide = WEIGHT && t > 0;
    const uint16_t lo = wide ? f32_to_e5m2x2(r[0], r[1]) : f32_to_e4m3x2(r[0], r[1]);
    const uint16_t hi = wide ? f32_to_e5m2x2(r[2], r[3]) : f32_to_e4m3x2(r[2], r[3]);
    part[t] = join16(lo, hi);
    if (t + 1 < T) {
      const uint32_t a = wide ? e5m2x2_to_f16x2(lo) : e4m3x2_to_f16x2(lo);
      const uint32_t b = wide ? e5m2x2_to_f16x2(hi) : e4m3x2_to_f16x2(hi);
      const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
      const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
      fma_pair(fa.x, fa.y, -1.f, -1.f, r[0], r[1], r[0], r[1]);
      fma_pair(fb.x, fb.y, -1.f, -1.f, r[2], r[3], r[2], r[3]);
      if (!WEIGHT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] *= 16.f;
      }
    }
  }
}
// The same for weights in two parts, by way of fp16: its 11 bits hold what
// the two parts (8 bits) can.
__device__ __forceinline__ void split4_f16(const float (&x)[4], uint32_t (&part)[2]) {
  const uint32_t a = pack_f16x2(x[0], x[1]), b = pack_f16x2(x[2], x[3]);
  const uint16_t a1 = f16x2_to_e4m3x2(a), b1 = f16x2_to_e4m3x2(b);
  part[0] = join16(a1, b1);
  const uint16_t a2 = f16x2_to_e5m2x2(sub_f16x2(a, e4m3x2_to_f16x2(a1)));
  const uint16_t b2 = f16x2_to_e5m2x2(sub_f16x2(b, e4m3x2_to_f16x2(b1)));
  part[1] = join16(a2, b2);
}

template <typename E>
__device__ __forceinline__ void unpack4(const uint2 raw, float (&x)[4]) {
  if constexpr (std::is_same<E, __nv_bfloat16>::value) {
    x[0] = __uint_as_float(raw.x << 16);
    x[1] = __uint_as_float(raw.x & 0xffff0000u);
    x[2] = __uint_as_float(raw.y << 16);
    x[3] = __uint_as_float(raw.y & 0xffff0000u);
  } else {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
  }
}

// The bf16 parts of a query by way of fp16 pairs: a scaled bf16 number's 8 bits
// and what the first part leaves of them are exact there.
__device__ __forceinline__ void split_query4(const float (&x)[4], uint32_t (&part)[2]) {
  const uint32_t a = pack_f16x2(x[0], x[1]), b = pack_f16x2(x[2], x[3]);
  const uint16_t a1 = f16x2_to_e4m3x2(a), b1 = f16x2_to_e4m3x2(b);
  part[0] = join16(a1, b1);
  const uint16_t a2 = f16x2_to_e4m3x2(mul16_f16x2(sub_f16x2(a, e4m3x2_to_f16x2(a1))));
  const uint16_t b2 = f16x2_to_e4m3x2(mul16_f16x2(sub_f16x2(b, e4m3x2_to_f16x2(b1))));
  part[1] = join16(a2, b2);
}

// The largest magnitude of four numbers, as the bits of a float's magnitude
// (which order like unsigned integers, NaN last).
template <typename E>
__device__ __forceinline__ uint32_t magnitude4(const uint2 raw) {
  const uint32_t a = raw.x & 0x7fff7fffu, b = raw.y & 0x7fff7fffu;
  const uint32_t m = __vmaxu2(a, b);
  const uint32_t most = max(m & 0xffffu, m >> 16);  // the type's own bits order the same way
  if constexpr (std::is_same<E, __nv_bfloat16>::value) return most << 16;
  if (most >= 0x7c00u) return 0x7f800000u;
  const __half h = *reinterpret_cast<const __half*>(&most);
  return __float_as_uint(__half2float(h));
}

// Sums each of a thread's N columns over the warp: lane c gets column c mod N.
// Each step adds up half of the columns with the lane across and gives the
// other half away.
template <int N>
__device__ __forceinline__ float sum_columns(float (&x)[N], int lane) {
#pragma unroll
  for (int half = N / 2; half > 0; half >>= 1) {
    const bool upper = (lane & half) != 0;
#pragma unroll
    for (int c = 0; c < half; ++c) {
      const float keep = upper ? x[c + half] : x[c], give = upper ? x[c] : x[c + half];
      x[c] = keep + __shfl_xor_sync(kAllLanes, give, half);
    }
  }
  float y = x[0];
#pragma unroll
  for (int d = N; d < 32; d <<= 1) y += __shfl_xor_sync(kAllLanes, y, d);
  return y;
}

// 2^x in two factors, since R may lie further below Q than float32 goes: the
// first is 1 down to x = -60.
__device__ __forceinline__ float2 exp2_factors(float x) {
  const bool far = x < -60.f;
  const float y = exp2_approx(far ? 0.5f * x : x);
  return make_float2(far ? y : 1.f, y);
}

// One work item's share of a rank.
struct Work {
  QuerySpan span;
  KeyList keys;
  int32_t kv, block;
  int32_t tiles, begin, steps;  // of the item; this rank's first and number
};

__device__ __forceinline__ Work find_work(const AttendArgs& a, const AttendPlan& plan, uint32_t unit, uint32_t rank,
                                          uint32_t ranks) {
  Work w;
  w.block = unit % plan.blocks;
  unit /= plan.blocks;
  w.kv = unit % a.cache.kv_heads;
  const int32_t item = unit / a.cache.kv_heads;
  w.span = QuerySpan{item, 1, 0, 0};
  w.keys = KeyList{};
  if (a.slots != nullptr) {
    w.keys = selected_keys(a, item);
  } else {
    w.span = find_span(a, item, plan.per);
    if (w.span.count > 0) w.keys = window_keys(a, w.span);
  }
  w.tiles = (w.keys.n + kTile - 1) / kTile;
  w.begin = static_cast<int32_t>(static_cast<int64_t>(w.tiles) * rank / ranks);
  w.steps = static_cast<int32_t>(static_cast<int64_t>(w.tiles) * (rank + 1) / ranks) - w.begin;
  return w;
}

// A column of an item: which of its queries, and which head.
struct Column {
  int32_t query, head;
  bool used;
};

template <int NH>
__device__ __forceinline__ Column find_column(const AttendArgs& a, const AttendPlan& plan, int32_t count, int32_t kv,
                                              int32_t block, int32_t c) {
  Column r;
  r.query = plan.per.divisor == 1 ? 0 : static_cast<int32_t>(fastdiv(c, plan.group));
  const int32_t g = c - r.query * a.heads_per_kv + block * NH;
  r.head = kv * a.heads_per_kv + g;
  r.used = r.query < count && g < a.heads_per_kv && (plan.per.divisor == 1 || block == 0);
  return r;
}

template <CacheShape SHAPE, int NH, int T>
__global__ void __launch_bounds__(Config<SHAPE, NH, T>::kThreads, 1)
    attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ AttendPlan plan) {
  using C = Config<SHAPE, NH, T>;
  using E = typename std::conditional<T == 2, __nv_bfloat16, __half>::type;
  using S = Shared<C, NH>;
  static_assert(C::kOffMisc + sizeof(S) <= C::kPipeBytes, "shared state");
  extern __shared__ __align__(1024) uint8_t all_smem[];
  const int lane = threadIdx.x & 31;
  const int pipe = C::kPipes == 1 ? 0 : __shfl_sync(kAllLanes, threadIdx.x / (C::kPipeWarps * 32), 0);
  const int tid = threadIdx.x - pipe * (C::kPipeWarps * 32);
  const int warp = __shfl_sync(kAllLanes, tid >> 5, 0);  // within the pipeline
  uint8_t* const smem = all_smem + pipe * C::kPipeBytes;
  const uint32_t base = smem_addr(smem);
  S& sh = *reinterpret_cast<S*>(smem + C::kOffMisc);
  constexpr int kLoadWarp = C::kSoftmax / 32;
  constexpr int kSplitWarp = kLoadWarp + C::kLoaders;
  constexpr int kMmaWarp = C::kPipeWarps - 1;
  // Named barriers: one for each softmax group, one for them all.
  constexpr int kFirstGroup = 1 + C::kPipes;

  // ---- set up, before the previous grid's results are needed
  if (tid == 0) {
    for (int c = 0; c < C::kLoadChunks; ++c) {
      for (int b = 0; b < C::kStages; ++b) {
        mbar_init(smem_addr(&sh.full[c][b]), C::kLoaders * (c == C::kNoteChunk ? 64 : 32));
        mbar_init(smem_addr(&sh.empty[c][b]), 1);
      }
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_addr(&sh.scores[b]), 1);
      mbar_init(smem_addr(&sh.queries[b]), C::kSplitters * 32);
      mbar_init(smem_addr(&sh.finished[b]), C::kSoftmax);
    }
    mbar_init(smem_addr(&sh.weights), C::kSoftmax);
    mbar_init(smem_addr(&sh.done), 1);
    mbar_init(smem_addr(&sh.queries_read), 1);
    mbar_init(smem_addr(&sh.drained), 1);
    sh.abort = a.wait_cycles == 0 ? 1 : 0;
    sh.last_known = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (tid < NH) {
    sh.best[0][tid] = ordered(-INFINITY);
    sh.reference[tid] = 5.f;
  }
  if (tid < C::kGroups) sh.unusual[tid] = 0;
  S& first = *reinterpret_cast<S*>(all_smem + C::kOffMisc);
  if (pipe == 0 && warp == kMmaWarp) tmem_alloc(smem_addr(&first.tmem), C::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_all = __shfl_sync(kAllLanes, first.tmem, 0);
  const uint32_t tmem = tmem_all + pipe * C::kPipeColumns;
  volatile int* abort = &sh.abort;
  // A wait's bound is one tile's, but for a wait that lasts over an item's tiles
  // or over the empty items before the next one.
  const int64_t bound = a.wait_cycles;
  pdl_wait();
  pdl_launch_dependents();

  // ---- this pipeline's items: whole ones, then perhaps a rank's share of one
  const uint32_t ctas = cluster_size();
  const uint32_t rank = cluster_ctarank() * C::kPipes + pipe, ranks = ctas * C::kPipes;
  const uint32_t whole_step = gridDim.x * C::kPipes;
  const int64_t item_bound = bound * (1 + plan.units / whole_step);
  const uint32_t split_unit = plan.whole + blockIdx.x / ctas;
  const bool has_split = split_unit < plan.units;
  // Softmax state that outlives the loop for a split item.
  float l[16];
  float reference = -INFINITY;  // R of column `own`

  if (warp < kLoadWarp) {
    // ==================================================== softmax
    const int wg = warp >> 2, thread = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // TMEM lane quadrant, << 16
    const int first_col = wg * 16;
    const int own = lane & 15;  // the column whose reference a lane keeps
    const int group_barrier = kFirstGroup + pipe * C::kGroups + wg;
    uint32_t n = 0, n3 = 0, b = 0, turn = 0;  // tiles so far; modulo 3; stage and its turn
    for (uint32_t seq = 0;; ++seq) {
      warp_wait(&sh.queries[seq & 1], (seq >> 1) & 1, abort, item_bound);
      // Everybody stops or nobody: the groups' barriers count on it.
      if (named_barrier_or(1 + pipe, C::kSoftmax, *abort != 0)) break;
      const Handed h = sh.handed[seq & 1];
      if (h.steps < 0) break;
      const bool several = h.count > 1;  // columns see different keys
      const int32_t all_to = h.position + 1;  // positions below are seen by every query, from
      const int32_t all_from =
          a.window == 0 ? 0 : static_cast<int32_t>(max(int64_t{0}, static_cast<int64_t>(h.position) + h.count - a.window));
#pragma unroll
      for (int c = 0; c < 16; ++c) l[c] = 0.f;
      reference = -INFINITY;
      float highest = -INFINITY;
      float t[16];              // a tile's scores, then u
      bool valid;               // this thread's key of it: whether it counts,
      float vs, scale, shift;   // its values' scale, the one used, its logarithm
      float top;                // column own's largest u
      float own_reference;      // Q of column own, where it is the warp's own
      // A tile up to its columns' maxima.
      auto begin_tile = [&]() {
        warp_wait(&sh.scores[n & 1], (n >> 1) & 1, abort, bound);
        tc_fence_after();
        const uint32_t s_at = tmem + lanes + C::kValues * NH + (n & 1) * (T * NH) + first_col;
        float s1[16];
        tmem_ld16(s_at, t);
        tmem_ld16(s_at + NH, s1);
        warp_wait(&sh.full[C::kNoteChunk][b], turn, abort, bound);
        valid = (sh.valid[b][warp & 3] >> lane) & 1;
        const float ks = sh.k_scale[b][thread];
        vs = C::kIsLatent ? ks : sh.v_scale[C::kIsLatent ? 0 : b][C::kIsLatent ? 0 : thread];
        if constexpr (T == 3) {
          float s2[16];
          tmem_ld16(s_at + 2 * NH, s2);
          tmem_wait_ld(t);
          tmem_wait_ld(s1);
          tmem_wait_ld(s2);
#pragma unroll
          for (int c = 0; c < 16; c += 2) fma_pair(s2[c], s2[c + 1], 0.0625f, 0.0625f, s1[c], s1[c + 1], s1[c], s1[c + 1]);
        } else {
          tmem_wait_ld(t);
          tmem_wait_ld(s1);
        }
        // u = log2(p) + log2(vscale): where the key is masked, -inf.
        scale = vs > 0.f ? fminf(fmaxf(vs, 0x1p-100f), 0x1p+100f) : vs == 0.f ? 0x1p-100f : vs;  // NaN stays
        shift = valid ? __log2f(scale) : -INFINITY;
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&sh.factor[seq & 1][first_col + c]);
          float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            mul_pair(fs[k], fs[k + 1], ks, ks, fs[k], fs[k + 1]);
            fma_pair(s1[c + k], s1[c + k + 1], 0.0625f, 0.0625f, t[c + k], t[c + k + 1], t[c + k], t[c + k + 1]);
            fma_pair(t[c + k], t[c + k + 1], fs[k], fs[k + 1], shift, shift, t[c + k], t[c + k + 1]);
          }
        }
        if constexpr (C::kSeveral) {
          if (several) {
            // The key is seen by the queries from its own position on, in a window
            // by the next window - 1 as well, or as a sink by all after it: a run
            // of the columns.
            const int32_t at = sh.position[b][thread];
            const bool sink = a.window == 0 || static_cast<uint32_t>(at) < a.sinks;
            if (!(at < all_to && (at >= all_from || sink))) {
              const int64_t ahead = static_cast<int64_t>(at) - h.position;  // the first query that sees it
              const int32_t from = static_cast<int32_t>(min(max(ahead, int64_t{0}), int64_t{NH})) * a.heads_per_kv;
              const int32_t to = sink ? NH : static_cast<int32_t>(min(max(ahead + a.window, int64_t{0}), int64_t{NH})) * a.heads_per_kv;
              const uint32_t seen = (0xffffu << min(max(from - first_col, 0), 16)) &
                                    ~(0xffffu << min(max(to - first_col, 0), 16));
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                if (!((seen >> c) & 1)) t[c] = -INFINITY;
              }
            }
          }
        }
        // Largest u of each column: lane c of a warp has column c's.
        top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float m = warp_max(t[c]);
          if (own == c) top = m;
        }
        int32_t* best = sh.best[n3];
        n3 = n3 == 2 ? 0 : n3 + 1;
        if (lane < 16) {
          atomicMax(&best[first_col + lane], ordered(top));
          if ((warp & 3) == 0) sh.best[n3][first_col + lane] = ordered(-INFINITY);
        }
        if (valid && !(fabsf(shift) <= kUsual)) sh.unusual[wg] = seq + 1;
        named_barrier(group_barrier, 128);
        top = unordered(best[first_col + own]);
      };
      // The rest, with the sum's reference R, or (APART) one of the warp's own.
      // False, and nothing done, where it has to be the latter.
      auto end_tile = [&](int32_t i, auto apart_tag) {
        constexpr bool APART = decltype(apart_tag)::value;
        if (!APART && __any_sync(kAllLanes, sh.unusual[wg] == seq + 1)) return false;
        const bool move = top > reference + 3.5f || (top < reference - 4.f && top > highest - 60.f);
        bool waited = i == 0;  // an item's end waits for its last outputs
        if (__any_sync(kAllLanes, move)) {
          const float to = move ? fmaxf(top, highest - 60.f) : reference;
          const float by = !move ? 1.f : reference == -INFINITY ? 0.f : exp2_approx(reference - to);
          reference = to;
          highest = fmaxf(highest, to);
          // The group's warps all write the same numbers: whoever reads them has
          // written them, and nobody is still at the tile before.
          if (lane < 16) sh.reference[first_col + lane] = to == -INFINITY ? 0.f : 5.f - to;
          __syncwarp();
          if (!waited) warp_wait(&sh.done, (n - 1) & 1, abort, bound);
          waited = true;
          tc_fence_after();
          float f[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            f[c] = __shfl_sync(kAllLanes, by, c);
            if (!APART) l[c] *= f[c];
          }
          if (i > 0) {
#pragma unroll 1
            for (int m = 0; m < C::kValues; ++m) {
              const uint32_t at = tmem + lanes + m * NH + first_col;
              float o[16];
              tmem_ld16(at, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] *= f[c];
              tmem_st16(at, o);
            }
            tmem_wait_st();
          }
        }
        if constexpr (APART) {
          const float back = valid && shift == shift ? shift : 0.f;  // u is -inf or NaN by itself
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float s = t[c] - back, most = warp_max(s);
            float q = __shfl_sync(kAllLanes, own_reference, c);
            if (most > q) {
              l[c] *= q == -INFINITY ? 1.f : exp2_approx(q - most);
              q = most;
              if (own == c) own_reference = q;
            }
            l[c] += exp2_approx(q == -INFINITY ? s : s - q);
          }
        }
        // Weights x = 2^(u - R + 5). The sum takes them in float32, without the
        // value's scale; the tensor core in T parts.
        const float to_sum = __fdividef(0.03125f, scale);
        const bool dead = vs == 0.f;  // values that count as 0, whatever their codes
        uint32_t part[4][T];
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          const float4 r = *reinterpret_cast<const float4*>(&sh.reference[first_col + c]);
          const float rs[4] = {r.x, r.y, r.z, r.w};
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            add_pair(t[c + k], t[c + k + 1], rs[k], rs[k + 1], x[k], x[k + 1]);
            x[k] = exp2_approx(x[k]);
            x[k + 1] = exp2_approx(x[k + 1]);
            if (!APART) fma_pair(x[k], x[k + 1], to_sum, to_sum, l[c + k], l[c + k + 1], l[c + k], l[c + k + 1]);
          }
          if constexpr (T == 2) {
            split4_f16(x, part[c / 4]);
          } else {
            split4<T, true>(x, part[c / 4]);
          }
        }
        if (dead) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int p = 0; p < T; ++p) part[c][p] = 0;
          }
        }
        if (!waited) warp_wait(&sh.done, (n - 1) & 1, abort, bound);
        const uint32_t at = NH == 64 ? thread * 64 + ((wg ^ ((thread >> 1) & 3)) << 4)
                            : NH == 32 ? thread * 32 + ((wg ^ ((thread >> 2) & 1)) << 4) : thread * 16;
#pragma unroll
        for (int p = 0; p < T; ++p) {
          st_shared_v4(base + C::kOffP + p * (NH * kTile) + at, part[0][p], part[1][p], part[2][p], part[3][p]);
        }
        fence_proxy_async();
        tc_fence_before();
        mbar_arrive(smem_addr(&sh.weights));
        ++n;
        if (++b == C::kStages) {
          b = 0;
          turn ^= 1;
        }
        return true;
      };
      int32_t i = 0;
      bool apart = false;
      for (; i < h.steps; ++i) {
        begin_tile();
        if (!end_tile(i, std::false_type{})) {
          apart = true;
          break;
        }
      }
      if (apart) {  // from here on all of the group's warps are
        own_reference = reference;
        while (true) {
          end_tile(i, std::true_type{});
          if (++i == h.steps) break;
          begin_tile();
        }
        // One reference for the item's end: 2^32 above the largest Q of the
        // warps, so that O fits as well, whatever the scales and the keys.
        warp_wait(&sh.done, (n - 1) & 1, abort, bound);
        tc_fence_after();
        float* qs = reinterpret_cast<float*>(smem + C::kOffP + wg * 4096) + 64;
        if (lane < 16) qs[(warp & 3) * 16 + lane] = own_reference;
        named_barrier(group_barrier, 128);
        float to = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) to = fmaxf(to, qs[w * 16 + own] + 32.f);
        // (Without a reference, a sum is 0 or not a number, and so are the outputs.)
        const float by = own_reference == -INFINITY ? 1.f : exp2_approx(own_reference - to);
        const float2 down = reference == -INFINITY ? make_float2(1.f, 1.f) : exp2_factors(reference - to);
        reference = to;
#pragma unroll
        for (int c = 0; c < 16; ++c) l[c] *= __shfl_sync(kAllLanes, by, c);
#pragma unroll 1
        for (int m = 0; m < C::kValues; ++m) {
          const uint32_t at = tmem + lanes + m * NH + first_col;
          float o[16];
          tmem_ld16(at, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = o[c] * __shfl_sync(kAllLanes, down.x, c) * __shfl_sync(kAllLanes, down.y, c);
          tmem_st16(at, o);
        }
        tmem_wait_st();
      }
      if (h.steps > 0) warp_wait(&sh.done, (n - 1) & 1, abort, bound);
      tc_fence_after();
      // Sums over the keys: lanes first, then the group's warps. The weights'
      // buffer is free by now and takes the warps' sums, then the outputs.
      float* sums = reinterpret_cast<float*>(smem + C::kOffP + wg * 4096);
      const float part_l = sum_columns(l, lane);
      if (lane < 16) sums[(warp & 3) * 16 + lane] = part_l;
      named_barrier(group_barrier, 128);
      l[0] = (sums[own] + sums[16 + own]) + (sums[32 + own] + sums[48 + own]);  // column own's
      if (h.split) break;
      const float inverse = l[0] == 0.f ? 0.f : 1.f / (32.f * l[0]);
      const bool failed = __any_sync(kAllLanes, *abort != 0);
      if ((warp & 3) == 0 && lane < 16 && !failed) {
        const Column col = find_column<NH>(a, plan, h.count, h.kv, h.block, first_col + lane);
        if (col.used) {
          a.lse[static_cast<int64_t>(h.row + col.query) * a.heads + col.head] =
              l[0] == 0.f ? -INFINITY : (reference + log2f(l[0])) * 0.69314718055994531f;
        }
      }
      named_barrier(group_barrier, 128);  // the sums are read
      // Outputs: a tile of 128 (D 64: 64) by 16 columns at a time through shared
      // memory, then in rows of a column.
      constexpr int kRowsOf = SHAPE == kDim64 ? 64 : 128;  // of M = 128
      constexpr int kPieces = kRowsOf / 8;                 // of 16 bytes in a row
      constexpr int kTurns = kPieces * 16 / 128;
      E* staged = reinterpret_cast<E*>(smem + C::kOffP + wg * 4096);
      E* out[kTurns];
#pragma unroll
      for (int k = 0; k < kTurns; ++k) {
        const int p = thread + k * 128;
        const Column col = find_column<NH>(a, plan, h.count, h.kv, h.block, first_col + p / kPieces);
        out[k] = !col.used || failed ? nullptr
                                     : static_cast<E*>(a.out) + static_cast<int64_t>(h.row + col.query) * a.out_row +
                                           static_cast<int64_t>(col.head) * a.out_head + p % kPieces * 8;
      }
      float inv[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) inv[c] = __shfl_sync(kAllLanes, inverse, c);
#pragma unroll 1
      for (int m = 0; m < C::kValues; ++m) {
        float o[16];
        if ((warp & 3) * 32 < kRowsOf) {
          tmem_ld16(tmem + lanes + m * NH + first_col, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            staged[c * 128 + thread] = static_cast<E>(o[c] * inv[c]);
          }
        }
        named_barrier(group_barrier, 128);
#pragma unroll
        for (int k = 0; k < kTurns; ++k) {
          const int p = thread + k * 128;
          const uint4 x = *reinterpret_cast<const uint4*>(staged + p / kPieces * 128 + p % kPieces * 8);
          if (out[k] != nullptr) {
            if (a.out_wide) {
              *reinterpret_cast<uint4*>(out[k] + m * 128) = x;
            } else {
              const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint16_t half = static_cast<uint16_t>(words[e / 2] >> (16 * (e & 1)));
                reinterpret_cast<uint16_t*>(out[k] + m * 128)[e] = half;
              }
            }
          }
        }
        if (m + 1 < C::kValues) named_barrier(group_barrier, 128);
      }
      // The next item's weights may overwrite any group's part of the buffer,
      // its outputs these.
      named_barrier(1 + pipe, C::kSoftmax);
      tc_fence_before();
      mbar_arrive(smem_addr(&sh.finished[seq & 1]));
    }
    tc_fence_before();
  } else if (warp < kSplitWarp) {
    // ==================================================== gathering
    // A warp gathers its share of a tile's 128 rows; lane r knows the places
    // of rows r, r + 32, ... (-1: masked, filled with zeros), eight lanes copy
    // a 128-byte row, four a 64-byte one. All places come round before the
    // first copy, so that the copies follow one another without a wait.
    constexpr int kShare = kTile / C::kLoaders;  // rows of a warp
    constexpr int kOwn = kShare / 32;            // rows whose place a lane knows
    constexpr int kLanes = C::kWide / 16;        // lanes to a main row
    constexpr int kRows = 32 / kLanes;           // rows at once
    constexpr int kTurns = kShare / kRows;       // turns for a warp's rows
    const int w = warp - kLoadWarp;
    const int sub = lane / kLanes;
    // Swizzled place of a lane's 16 bytes, in even and odd turns.
    const uint32_t in_even = C::kWide == 128 ? ((lane ^ sub) & 7) << 4 : ((lane ^ (sub >> 1)) & 3) << 4;
    const uint32_t in_odd = C::kWide == 128 ? ((lane ^ (sub + 4)) & 7) << 4 : in_even;
    const bool alike = a.cache.k_block_rows == a.cache.v_block_rows && a.cache.k_token_rows == a.cache.v_token_rows &&
                       a.cache.k_head_rows == a.cache.v_head_rows;
    bool bad = false;
    uint32_t b = 0, turn = 0, tail_turn = 0;
    uint32_t unit = blockIdx.x * C::kPipes + pipe;
    bool shared = false;  // at the split item
    while (true) {
      Work work;
      if (unit < plan.whole) {
        work = find_work(a, plan, unit, 0, 1);
        unit += whole_step;
      } else if (has_split && !shared) {
        work = find_work(a, plan, split_unit, rank, ranks);
        shared = true;
      } else {
        break;
      }
      const uint32_t k_first = work.kv * a.cache.k_head_rows, v_first = work.kv * a.cache.v_head_rows;
      const int32_t mine = work.begin * kTile + w * kShare + lane;
      int32_t fetched[kOwn];  // slots or table entries, a tile ahead
#pragma unroll
      for (int o = 0; o < kOwn; ++o) fetched[o] = work.steps > 0 ? fetch_key(a, work.keys, mine + o * 32) : -1;
      for (int32_t i = 0; i < work.steps; ++i) {
        int32_t k_row[kOwn], v_row[kOwn], position[kOwn];
        uint32_t page[kOwn];
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
          const int32_t j = mine + i * kTile + o * 32;
          const Key key = locate_key(a, work.keys, j, fetched[o]);
          bad |= bad_key(work.keys, j, fetched[o], key);
          fetched[o] = fetch_key(a, work.keys, j + kTile);
          page[o] = key.block;
          position[o] = key.position;
          k_row[o] = key.valid ? static_cast<int32_t>(k_first + key.block * a.cache.k_block_rows + key.offset * a.cache.k_token_rows) : -1;
          v_row[o] = key.valid ? static_cast<int32_t>(v_first + key.block * a.cache.v_block_rows + key.offset * a.cache.v_token_rows) : -1;
        }
        int32_t row[kTurns];
#pragma unroll
        for (int n = 0; n < kTurns; ++n) {
          row[n] = __shfl_sync(kAllLanes, k_row[n * kRows / 32], (n * kRows) % 32 + sub);
        }
        // Copies `kWide` bytes of every row, from column x on, to a chunk.
        auto copy = [&](uint32_t to, const uint8_t* from, int64_t pitch) {
          to += (w * kShare + sub) * C::kWide;
          from += (lane % kLanes) * 16;
#pragma unroll
          for (int n = 0; n < kTurns; ++n) {
            cp_async16(to + n * kRows * C::kWide + (n & 1 ? in_odd : in_even), from + max(row[n], 0) * pitch,
                       row[n] < 0 ? 0 : 16);
          }
        };
        // What the softmax has to know of a key: copied with its tile.
        auto note = [&]() {
#pragma unroll
          for (int o = 0; o < kOwn; ++o) {
            const int at = w * kShare + o * 32 + lane;
            const int64_t scale_at = static_cast<int64_t>(page[o]) * a.cache.kv_heads + work.kv;
            const uint32_t size = k_row[o] < 0 ? 0 : 4;
            cp_async4(smem_addr(&sh.k_scale[b][at]), a.cache.k_scale + scale_at, size);
            if constexpr (!C::kIsLatent) cp_async4(smem_addr(&sh.v_scale[b][at]), a.cache.v_scale + scale_at, size);
            if constexpr (C::kSeveral) sh.position[b][at] = position[o];
            const uint32_t valid = __ballot_sync(kAllLanes, k_row[o] >= 0);
            if (lane == 0) sh.valid[b][w * kOwn + o] = valid;
          }
          mbar_arrive(smem_addr(&sh.full[C::kNoteChunk][b]));
        };
        const uint32_t stage = base + b * C::kStageBytes;
        if constexpr (C::kIsLatent) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            warp_wait(&sh.empty[c][b], turn ^ 1, abort, bound);
            copy(stage + c * C::kChunkBytes, a.cache.k + c * 128, a.cache.k_pitch);
            if (c == C::kNoteChunk) note();
            cp_async_arrive(smem_addr(&sh.full[c][b]));
          }
          const uint32_t tb = C::kTails == 1 ? 0 : b, tt = C::kTails == 1 ? tail_turn : turn;
          tail_turn ^= 1;
          warp_wait(&sh.empty[4][tb], tt ^ 1, abort, bound);
          const uint32_t to = base + C::kOffTail + tb * C::kTailBytes + (w * kShare + lane / 4) * 64 +
                              (((lane ^ (lane >> 3)) & 3) << 4);
#pragma unroll
          for (int n = 0; n < kShare / 8; ++n) {
            const int32_t r = __shfl_sync(kAllLanes, k_row[n * 8 / 32], (n * 8) % 32 + lane / 4);
            cp_async16(to + n * 512, a.cache.k + 512 + (lane % 4) * 16 + max(r, 0) * a.cache.k_pitch, r < 0 ? 0 : 16);
          }
          cp_async_arrive(smem_addr(&sh.full[4][tb]));
        } else {
          // 64-byte rows: values first, so that their second half of M reads
          // the keys behind them.
          const uint32_t keys_at = stage + (SHAPE == kDim64 ? C::kChunkBytes : 0);
          const uint32_t values_at = stage + (SHAPE == kDim64 ? 0 : C::kChunkBytes);
          warp_wait(&sh.empty[0][b], turn ^ 1, abort, bound);
          copy(keys_at, a.cache.k, a.cache.k_pitch);
          cp_async_arrive(smem_addr(&sh.full[0][b]));
          if (!alike) {
#pragma unroll
            for (int n = 0; n < kTurns; ++n) {
              row[n] = __shfl_sync(kAllLanes, v_row[n * kRows / 32], (n * kRows) % 32 + sub);
            }
          }
          warp_wait(&sh.empty[1][b], turn ^ 1, abort, bound);
          copy(values_at, a.cache.v, a.cache.v_pitch);
          note();
          cp_async_arrive(smem_addr(&sh.full[1][b]));
        }
        if (++b == C::kStages) {
          b = 0;
          turn ^= 1;
        }
        if (__any_sync(kAllLanes, *abort != 0)) break;
      }
      if (__any_sync(kAllLanes, *abort != 0)) break;
    }
    cp_async_wait_all();
    if (__any_sync(kAllLanes, bad) && lane == 0) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
  } else if (warp < kMmaWarp) {
    // ==================================================== queries
    // Find the next item, bring its queries, split them as soon as the last
    // scores of the item before are done, and hand it on. Items without keys
    // end here: out 0, lse -inf.
    const int w = warp - kSplitWarp;
    uint32_t unit = blockIdx.x * C::kPipes + pipe, seq = 0;
    int32_t steps_before = 0;  // tiles of the item before
    bool shared = false;
    while (true) {
      Work work;
      bool end = false;
      const bool split = unit >= plan.whole;
      if (!split) {
        work = find_work(a, plan, unit, 0, 1);
        unit += whole_step;
      } else if (has_split && !shared) {
        work = find_work(a, plan, split_unit, rank, ranks);
        shared = true;
        if (w == 0 && lane == 0) {
          sh.last = Handed{work.span.row, work.span.count, work.span.position, work.kv, work.block, work.steps,
                           work.tiles > 0 ? 1 : 0};
          sh.last_known = 1;
        }
      } else {
        end = true;
      }
      constexpr int kPieces = (C::kKeyDim / 4 + 31) / 32;
      constexpr int kBatch = 2;  // columns side by side: a column's own steps follow one another
      uint2 raw[kBatch][kPieces];
      auto bring = [&](int c0) {
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const Column col = find_column<NH>(a, plan, work.span.count, work.kv, work.block, c0 + n);
          const int64_t at = col.used ? static_cast<int64_t>(work.span.row + col.query) * a.q_row +
                                            static_cast<int64_t>(col.head) * a.q_head : 0;
          const E* q = static_cast<const E*>(a.q) + at + lane * 4;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            raw[n][i] = make_uint2(0u, 0u);
            if (col.used && (i * 32 + lane) * 4 < C::kKeyDim) raw[n][i] = ld_global_v2(q + i * 128);
          }
        }
      };
      if (!end) {
        if (work.tiles == 0) {
          if (!split || rank == 0) {
            for (int c = w; c < NH; c += C::kSplitters) {
              const Column col = find_column<NH>(a, plan, work.span.count, work.kv, work.block, c);
              if (!col.used) continue;
              const int64_t row = work.span.row + col.query;
              E* out = static_cast<E*>(a.out) + row * a.out_row + static_cast<int64_t>(col.head) * a.out_head;
              for (int d = lane; d < C::kValueDim; d += 32) out[d] = static_cast<E>(0.f);
              if (lane == 0) a.lse[row * a.heads + col.head] = -INFINITY;
            }
          }
          continue;
        }
        // Towards L2, while the item before still needs the buffer (unused
        // columns: the first row, so that the lanes stay together).
        for (int e = w * 32; e < NH * C::kKeyDim / 64; e += C::kSplitters * 32) {
          const int first = min(e + lane, NH * C::kKeyDim / 64 - 1) * 64;
          const Column col = find_column<NH>(a, plan, work.span.count, work.kv, work.block, first / C::kKeyDim);
          const int64_t at = col.used ? static_cast<int64_t>(work.span.row + col.query) * a.q_row +
                                            static_cast<int64_t>(col.head) * a.q_head + first % C::kKeyDim : 0;
          prefetch_l2_line(static_cast<const E*>(a.q) + at);
        }
        __syncwarp();
        bring(w * kBatch);
      }
      if (seq > 0) warp_wait(&sh.queries_read, (seq - 1) & 1, abort, bound * (steps_before + 1));
      if (seq > 1) warp_wait(&sh.finished[seq & 1], ((seq >> 1) - 1) & 1, abort, bound);
      if (__any_sync(kAllLanes, *abort != 0)) break;  // what was handed on stays
      if (end) {
        if (w == 0 && lane == 0) sh.handed[seq & 1].steps = -1;
        __syncwarp();
        mbar_arrive(smem_addr(&sh.queries[seq & 1]));
        break;
      }
      if (w == 0 && lane == 0) {
        sh.handed[seq & 1] = Handed{work.span.row, work.span.count, work.span.position, work.kv, work.block, work.steps,
                                    split ? 1 : 0};
      }
      for (int c0 = w * kBatch; c0 < NH; c0 += C::kSplitters * kBatch) {
        uint2 now[kBatch][kPieces];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
#pragma unroll
          for (int i = 0; i < kPieces; ++i) now[n][i] = raw[n][i];
        }
        if (c0 + C::kSplitters * kBatch < NH) bring(c0 + C::kSplitters * kBatch);  // the next ones come during these
        uint32_t most[kBatch];
        float up[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          most[n] = 0;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) most[n] = max(most[n], magnitude4<E>(now[n][i]));
        }
#pragma unroll
        for (int n = 0; n < kBatch; ++n) most[n] = __reduce_max_sync(kAllLanes, most[n]);
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          // The largest magnitude comes to [128, 256): its exponent field is taken off.
          const int e = max(static_cast<int>(most[n] >> 23), 40);
          const bool odd = most[n] >= 0x7f800000u;  // an infinity or NaN: the row becomes NaN
          up[n] = odd ? 0.f : __uint_as_float(static_cast<uint32_t>(134 + 127 - e) << 23);
          if (lane == n) sh.factor[seq & 1][c0 + n] = odd ? NAN : a.scale_log2 * __uint_as_float(static_cast<uint32_t>(e - 7) << 23);
        }
        __syncwarp();
        // A lane's four columns of piece i are bytes 4 lane on of chunk i; a
        // part's rows lie NH rows behind the part before.
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const bool narrow = C::kWide == 64 || (C::kIsLatent && i == 4);
#pragma unroll
          for (int n = 0; n < kBatch; ++n) {
            const int c = c0 + n;
            float y[4];
            unpack4<E>(now[n][i], y);
            mul_pair(y[0], y[1], up[n], up[n], y[0], y[1]);
            mul_pair(y[2], y[3], up[n], up[n], y[2], y[3]);
            uint32_t part[T];
            if constexpr (T == 2) {
              split_query4(y, part);
            } else {
              split4<T, false>(y, part);
            }
            const uint32_t at = base + C::kOffQ + (lane & 3) * 4 + i * (T * NH * 128) +
                                (narrow ? c * 64 + ((((lane >> 2) ^ (c >> 1)) & 3) << 4) : c * 128 + ((((lane >> 2) ^ c) & 7) << 4));
            if (!narrow || lane < 16) {
#pragma unroll
              for (int t = 0; t < T; ++t) st_shared(at + t * (NH * (narrow ? 64 : 128)), part[t]);
            }
          }
        }
      }
      fence_proxy_async();
      mbar_arrive(smem_addr(&sh.queries[seq & 1]));
      steps_before = work.steps;
      ++seq;
      if (split) break;
    }
  } else {
    // ==================================================== MMAs
    // The whole warp walks the loops, so that addresses stay in uniform
    // registers; one lane issues.
    constexpr uint32_t kScoreDesc = mma_descriptor(128, T * NH, kE4M3, false, false);
    constexpr uint32_t kFirstDesc = mma_descriptor(128, NH, kE4M3, true, true);
    constexpr uint32_t kOtherDesc = mma_descriptor(128, NH, kE5M2, true, true);
    constexpr Swizzle kPSwizzle = NH == 64 ? kSwizzle64 : NH == 32 ? kSwizzle32 : kSwizzleNone;
    constexpr Swizzle kMain = C::kWide == 128 ? kSwizzle128 : kSwizzle64;
    // Descriptors of the first chunks; further ones are offsets in units of 16 bytes.
    const uint64_t k_desc = smem_descriptor(base + (SHAPE == kDim64 ? C::kChunkBytes : 0), 16, 8 * C::kWide, kMain);
    const uint64_t q_desc = smem_descriptor(base + C::kOffQ, 16, 8 * C::kWide, kMain);
    const uint64_t v_desc = smem_descriptor(base + (SHAPE == kDim128 ? C::kChunkBytes : 0),
                                            SHAPE == kDim64 ? C::kChunkBytes : 1024, 8 * C::kWide, kMain);
    const uint64_t p_desc = smem_descriptor(base + C::kOffP, 8 * NH, 8 * NH, kPSwizzle);
    const bool leader = elect_one();
    uint32_t sb = 0, st = 0, ob = 0, ot = 0, tail_turn = 0;  // stage and its turn, of scores and of outputs
    uint32_t n = 0;                                          // tiles before this item
    bool more = true;
    for (uint32_t seq = 0; more; ++seq) {
      warp_wait(&sh.queries[seq & 1], (seq >> 1) & 1, abort, item_bound);
      if (__any_sync(kAllLanes, *abort != 0)) break;
      const int32_t steps = __shfl_sync(kAllLanes, sh.handed[seq & 1].steps, 0);
      more = steps >= 0 && __shfl_sync(kAllLanes, sh.handed[seq & 1].split, 0) == 0;
      auto scores = [&](int32_t i) {
        const uint32_t d = tmem + C::kValues * NH + ((n + i) & 1) * (T * NH);
#pragma unroll
        for (int c = 0; c < C::kMainKeys; ++c) {
          warp_wait(&sh.full[c][sb], st, abort, bound);
          fence_proxy_async();  // the copies wrote through the generic proxy
          if (leader) {
            const uint64_t kd = k_desc + ((sb * C::kStageBytes + c * C::kChunkBytes) >> 4);
            const uint64_t qd = q_desc + ((c * (T * NH * C::kWide)) >> 4);
#pragma unroll
            for (int k = 0; k < C::kWide / 32; ++k) mma_f8(d, kd + 2 * k, qd + 2 * k, kScoreDesc, c + k > 0);
          }
          __syncwarp();
        }
        if constexpr (C::kIsLatent) {
          const uint32_t tb = C::kTails == 1 ? 0 : sb, tt = C::kTails == 1 ? tail_turn : st;
          tail_turn ^= 1;
          warp_wait(&sh.full[4][tb], tt, abort, bound);
          fence_proxy_async();
          if (leader) {
            const uint64_t kd = smem_descriptor(base + C::kOffTail + tb * C::kTailBytes, 16, 512, kSwizzle64);
            const uint64_t qd = smem_descriptor(base + C::kOffQ + 4 * (T * NH * 128), 16, 512, kSwizzle64);
            mma_f8(d, kd, qd, kScoreDesc, true);
            mma_f8(d, kd + 2, qd + 2, kScoreDesc, true);
            mma_commit(smem_addr(&sh.empty[4][tb]));
          }
        } else if (leader) {
          mma_commit(smem_addr(&sh.empty[0][sb]));
        }
        if (leader) {
          mma_commit(smem_addr(&sh.scores[(n + i) & 1]));
          if (i + 1 == steps) mma_commit(smem_addr(&sh.queries_read));
        }
        __syncwarp();
        if (++sb == C::kStages) {
          sb = 0;
          st ^= 1;
        }
      };
      auto outputs = [&](int32_t i) {
        warp_wait(&sh.weights, (n + i) & 1, abort, bound);
        tc_fence_after();
        if constexpr (!C::kIsLatent) {
          warp_wait(&sh.full[1][ob], ot, abort, bound);
          fence_proxy_async();
        }
        if (leader) {
#pragma unroll
          for (int c = 0; c < C::kValues; ++c) {
            const uint64_t vd = v_desc + ((ob * C::kStageBytes + c * C::kChunkBytes) >> 4);
#pragma unroll
            for (int p = 0; p < T; ++p) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                mma_f8(tmem + c * NH, vd + 2 * C::kWide * k, p_desc + ((p * (NH * kTile) + k * 32 * NH) >> 4),
                       p == 0 ? kFirstDesc : kOtherDesc, p + k > 0 || i > 0);
              }
            }
            mma_commit(smem_addr(&sh.empty[C::kIsLatent ? c : 1][ob]));
          }
          mma_commit(smem_addr(&sh.done));
        }
        __syncwarp();
        if (++ob == C::kStages) {
          ob = 0;
          ot ^= 1;
        }
      };
      // Scores run a tile ahead of the outputs, so that a softmax overlaps the
      // next tile's scores.
#pragma unroll 1
      for (int32_t i = 0; i <= steps && steps > 0; ++i) {
        if (i < steps) scores(i);
        if (i > 0) outputs(i - 1);
        if (__any_sync(kAllLanes, *abort != 0)) break;
      }
      if (steps > 0) n += steps;
    }
    if (__any_sync(kAllLanes, *abort != 0)) {  // gave up: let what was issued finish before the memory goes
      if (leader) {
        mma_commit(smem_addr(&sh.drained));
        const long long begin = clock64();
        while (!mbar_try(smem_addr(&sh.drained), 0) && clock64() - begin < 4000000000LL) {
        }
        flag_status(a.status, SILKERN_STATUS_WAIT_TIMEOUT);
      }
      __syncwarp();
    }
  }

  __syncthreads();
  const bool gave_up = *abort != 0;
  // ---- a split item: its ranks, which all see the same tiles, join
  Handed last{};
  if (has_split) {
    if (sh.last_known != 0) {
      last = sh.last;
    } else {  // the query warps gave up before it
      const Work work = find_work(a, plan, split_unit, rank, ranks);
      last = Handed{work.span.row, work.span.count, work.span.position, work.kv, work.block, work.steps, work.tiles > 0 ? 1 : 0};
    }
  }
  if (last.split) {
    const uint32_t share = (NH + ranks - 1) / ranks;                    // columns of a rank at most
    float* joint = reinterpret_cast<float*>(smem + C::kOffP) + 8 * NH;  // references, then sums
    float* joined = reinterpret_cast<float*>(smem);                     // outputs: (rank, column of this rank, value)
    const int first_col = (warp >> 2) * 16, own = lane & 15;
    if (warp < kLoadWarp && (warp & 3) == 0 && lane < 16) {
      joint[first_col + lane] = reference;
      joint[NH + first_col + lane] = gave_up ? NAN : l[0];  // and so every rank's results
    }
    cluster_sync();
    // Rank r is pipeline r mod kPipes of CTA r / kPipes.
    const uint32_t origin = smem_addr(all_smem);
    auto place = [&](const float* p, uint32_t r) {
      return map_cluster(origin + (r % C::kPipes) * C::kPipeBytes + (smem_addr(p) - base), r / C::kPipes);
    };
    if (warp < kLoadWarp) {
      // A column's ranks, the even ones in one lane and the odd ones in another.
      const float* at = joint + first_col + own;
      constexpr int kHalf = C::kMostRanks / 2;
      float rr[kHalf], ll[kHalf];
#pragma unroll
      for (uint32_t k = 0; k < kHalf; ++k) {
        const uint32_t r = 2 * k + (lane >> 4);
        rr[k] = -INFINITY;
        ll[k] = 0.f;
        if (r < ranks) {
          rr[k] = ld_cluster(place(at, r));
          ll[k] = ld_cluster(place(at + NH, r));
        }
      }
      float whole_r = -INFINITY, whole_l = 0.f;
#pragma unroll
      for (uint32_t k = 0; k < kHalf; ++k) whole_r = fmaxf(whole_r, rr[k]);
      whole_r = fmaxf(whole_r, __shfl_xor_sync(kAllLanes, whole_r, 16));
#pragma unroll
      for (uint32_t k = 0; k < kHalf; ++k) {
        // (A rank without a reference saw nothing, or only what is not a number.)
        whole_l += rr[k] == -INFINITY ? ll[k] : ll[k] * exp2_approx(rr[k] - whole_r);
      }
      whole_l += __shfl_xor_sync(kAllLanes, whole_l, 16);
      const float inverse = whole_l == 0.f ? 0.f : 1.f / (32.f * whole_l);
      const float2 down = reference == -INFINITY ? make_float2(1.f, 0.f) : exp2_factors(reference - whole_r);
      const float by = down.y * inverse;
      const bool far = __any_sync(kAllLanes, down.x != 1.f);
      if (rank == 0 && (warp & 3) == 0 && lane < 16) {
        const Column col = find_column<NH>(a, plan, last.count, last.kv, last.block, first_col + lane);
        if (col.used) {
          a.lse[static_cast<int64_t>(last.row + col.query) * a.heads + col.head] =
              whole_l == 0.f ? -INFINITY : (whole_r + log2f(whole_l)) * 0.69314718055994531f;
        }
      }
      __syncwarp();
      tc_fence_after();
      // Rank r joins the columns from NH r / ranks to NH (r + 1) / ranks, and
      // gets every rank's part of them: stores need no answer, loads would wait
      // for one.
      const uint32_t joiner = ((first_col + own + 1) * ranks - 1) / NH;
      const uint32_t joined_at =
          place(joined + (rank * share + first_col + own - NH * joiner / ranks) * C::kValueDim, joiner);
      if (SHAPE != kDim64 || (warp & 3) < 2) {
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
#pragma unroll 1
        for (int m = 0; m < C::kValues; ++m) {
          float o[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = 0.f;
          if (last.steps > 0) {
            tmem_ld16(tmem + lanes + m * NH + first_col, o);
            tmem_wait_ld(o);
            if (far) {
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] *= __shfl_sync(kAllLanes, down.x, c);
            }
          }
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float f = __shfl_sync(kAllLanes, by, c);
            const uint32_t to = __shfl_sync(kAllLanes, joined_at, c);
            st_cluster(to + (m * 128 + (tid & 127)) * 4, last.steps > 0 ? o[c] * f : 0.f);
          }
        }
      }
    }
    cluster_sync();  // the last time that a CTA touches another's memory is before
    constexpr int kRankThreads = C::kPipeWarps * 32;
    const int32_t mine = NH * rank / ranks, joins = NH * (rank + 1) / ranks - mine;
    for (int32_t e = tid * 4; e < joins * C::kValueDim; e += kRankThreads * 4) {
      const int32_t c = e / C::kValueDim, d = e - c * C::kValueDim;
      const Column col = find_column<NH>(a, plan, last.count, last.kv, last.block, mine + c);
      if (!col.used) continue;
      float4 y{0.f, 0.f, 0.f, 0.f};
      for (uint32_t r = 0; r < ranks; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(joined + r * share * C::kValueDim + e);
        y.x += x.x;
        y.y += x.y;
        y.z += x.z;
        y.w += x.w;
      }
      E* out = static_cast<E*>(a.out) + static_cast<int64_t>(last.row + col.query) * a.out_row +
               static_cast<int64_t>(col.head) * a.out_head + d;
      out[0] = static_cast<E>(y.x);
      out[1] = static_cast<E>(y.y);
      out[2] = static_cast<E>(y.z);
      out[3] = static_cast<E>(y.w);
    }
    tc_fence_before();
    __syncthreads();
  }
  if (gave_up) {  // no result of this pipeline's items is left as it was before the call
    uint32_t unit = blockIdx.x * C::kPipes + pipe;
    bool rest = has_split && !last.split && rank == 0;  // a split item without keys
    while (unit < plan.whole || rest) {
      const bool whole = unit < plan.whole;
      const Work work = find_work(a, plan, whole ? unit : split_unit, 0, 1);
      unit = whole ? unit + whole_step : unit;
      rest = rest && whole;
      for (int c = warp; c < NH; c += C::kPipeWarps) {
        const Column col = find_column<NH>(a, plan, work.span.count, work.kv, work.block, c);
        if (!col.used) continue;
        const int64_t row = work.span.row + col.query;
        E* out = static_cast<E*>(a.out) + row * a.out_row + static_cast<int64_t>(col.head) * a.out_head;
        for (int d = lane; d < C::kValueDim; d += 32) out[d] = static_cast<E>(NAN);
        if (lane == 0) a.lse[row * a.heads + col.head] = NAN;
      }
    }
  }
  if (pipe == 0 && warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem_all, C::kColumns);
  }
}

template <CacheShape SHAPE, int NH, int T>
int launch_config(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  using C = Config<SHAPE, NH, T>;
  static DeviceBits granted{0};
  const int rc = allow_launch(reinterpret_cast<const void*>(attend_kernel<SHAPE, NH, T>), kSharedMemory, granted);
  if (rc != SILKERN_OK) return rc;
  return launch_pdl(attend_kernel<SHAPE, NH, T>, l.grid, C::kThreads, kSharedMemory, l.cluster, l.stream, a, plan);
}

template <CacheShape SHAPE>
int launch_shape(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  if (l.half) {
    if (l.columns == 16) return launch_config<SHAPE, 16, 3>(a, plan, l);
    if (l.columns == 32) return launch_config<SHAPE, 32, 3>(a, plan, l);
    if constexpr (SHAPE != kLatent) return launch_config<SHAPE, 64, 3>(a, plan, l);
    return SILKERN_E_GEOMETRY;
  }
  if (l.columns == 16) return launch_config<SHAPE, 16, 2>(a, plan, l);
  if (l.columns == 32) return launch_config<SHAPE, 32, 2>(a, plan, l);
  return launch_config<SHAPE, 64, 2>(a, plan, l);
}

}  // namespace silkern
