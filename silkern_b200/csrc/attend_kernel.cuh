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
// Weights: with u_j = log2(p_j) + log2(vscale_j) and R a reference near the
// tile's largest u, P'_j = 2^(u_j - R + 5) goes to the tensor core and
// 2^(log2 p_j - R) to the sum, so out = O / (32 l) and lse = (R + log2 l) ln 2
// hold for any scales in [2^-100, 2^100]. R moves, and O and l are rescaled,
// only when a tile's largest u leaves [R - 4, R + 3.5]: e4m3 ends at 448 =
// 2^8.8. l, S and O are float32.
//
// Warps: 4 or 8 for the softmax (one key each thread), 4 that gather keys and
// values with cp.async, one that issues the MMAs. Few work items are split
// over the keys by a thread-block cluster, whose CTAs join their sums and
// outputs through distributed shared memory: no workspace, one launch.
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
// A CTA's share of the 228 KB of an SM is at least its share of the 512 TMEM
// columns, 456 bytes a column with the 1 KB that the SM adds to each CTA. So
// CTAs of these kernels that fit an SM's shared memory also fit its TMEM, and
// none waits for TMEM that a member of another waiting cluster holds.
constexpr int smem_for_columns(int columns) { return columns * 456 - 1024; }

template <CacheShape SHAPE, int NH, int T>
struct Config {
  static constexpr bool kIsLatent = SHAPE == kLatent;
  static constexpr int kKeyDim = SHAPE == kDim64 ? 64 : SHAPE == kDim128 ? 128 : 576;
  static constexpr int kValueDim = SHAPE == kDim64 ? 64 : SHAPE == kDim128 ? 128 : 512;
  static constexpr int kWide = SHAPE == kDim64 ? 64 : 128;      // row bytes of the main chunks
  static constexpr int kMainKeys = kIsLatent ? 4 : 1;           // K chunks of kWide bytes
  static constexpr int kValues = kIsLatent ? 4 : 1;             // V chunks: M = 128 tiles of O^T
  static constexpr int kLoadChunks = kIsLatent ? 5 : 2;  // barriers: four wide chunks and the tail; else keys, values
  static constexpr int kChunkBytes = kWide * kTile;
  static constexpr int kStageBytes = (kIsLatent ? 4 : 2) * kChunkBytes;
  static constexpr int kTailBytes = kIsLatent ? 64 * kTile : 0;  // a latent key's last 64 bytes
  static constexpr int kGroups = NH >= 32 ? 2 : 1;               // softmax warpgroups, by columns
  static constexpr int kCols = NH / kGroups;                     // columns of a softmax thread
  static constexpr int kSoftmax = kGroups * 128;
  // Two CTAs to an SM where a column block is narrow: each hides the other's
  // start, end and softmax. With 4 + 2 + 1 warps (registers are given out for
  // eight) both have 128 registers a thread. Otherwise one CTA, with all of
  // shared memory.
  static constexpr int kPerSm = !kIsLatent && NH == 16 ? 2 : 1;
  static constexpr int kLoaders = kPerSm == 2 ? 2 : 4;           // gathering warps
  static constexpr int kThreads = kSoftmax + kLoaders * 32 + 32;
  static constexpr int kQBytes = T * NH * kKeyDim;
  static constexpr int kPBytes = T * NH * kTile;
  // Columns of several queries see different keys. 64 columns of a latent
  // cache are one query's, so that its shared memory need not hold positions.
  static constexpr bool kSeveral = !(kIsLatent && NH == 64);
  static constexpr int kNoteBytes = kTile * ((kIsLatent ? 4 : 8) + (kSeveral ? 4 : 0)) + 16;  // a tile's scales, positions
  static constexpr int kMisc = 20 * NH + (kSeveral ? 8 * NH : 0) + 256;
  static constexpr int kColumnsUsed = kValues * NH + 2 * T * NH;
  static constexpr int kColumns = kColumnsUsed <= 128 ? 128 : kColumnsUsed <= 256 ? 256 : 512;
  static_assert(kColumnsUsed <= 512, "TMEM");
  static constexpr int kSmemMax = smem_for_columns(512 / kPerSm);
  static constexpr int kFixed = kQBytes + kPBytes + kMisc;
  static constexpr int kStageCost = kStageBytes + kNoteBytes + 16 * kLoadChunks;  // with its barriers
  static constexpr int kFit = (kSmemMax - kFixed) / kStageCost;
  static constexpr int kStages = kIsLatent ? 2 : kFit < 8 ? kFit : 8;
  static constexpr int kTails = kIsLatent ? ((kSmemMax - kFixed - 2 * kStageCost) >= 2 * kTailBytes ? 2 : 1) : 0;
  static constexpr int kUsed = kFixed + kStages * kStageCost + kTails * kTailBytes;
  static_assert(kStages >= 2 && kUsed <= kSmemMax, "shared memory");
  static constexpr int kSmem = kUsed > smem_for_columns(kColumns) ? kUsed : smem_for_columns(kColumns);
  static_assert(NH * kValueDim * 4 <= kStages * kStageBytes, "joining buffer");
  // The chunk whose buffer is free again only after a tile's softmax, and
  // with it the tile's scales and positions.
  static constexpr int kNoteChunk = kIsLatent ? 0 : 1;
  // Offsets from the dynamic shared memory's start.
  static constexpr int kOffTail = kStages * kStageBytes;
  static constexpr int kOffQ = kOffTail + kTails * kTailBytes;
  static constexpr int kOffP = kOffQ + kQBytes;
  static constexpr int kOffMisc = kOffP + kPBytes;
};

// The small shared state behind the tiles.
template <typename C, int NH>
struct __align__(16) Shared {
  int32_t best[3][NH];  // column maxima of a tile, as ordered integers
  float reference[NH];  // the columns' references R, at the end their output factors
  float factor[NH];     // the columns' score factors
  int32_t seen_to[C::kSeveral ? NH : 1], seen_from[C::kSeveral ? NH : 1];  // positions that a column sees: below, from
  float k_scale[C::kStages][kTile];
  float v_scale[C::kIsLatent ? 1 : C::kStages][C::kIsLatent ? 1 : kTile];
  int32_t position[C::kSeveral ? C::kStages : 1][C::kSeveral ? kTile : 1];
  uint32_t valid[C::kStages][4];  // a bit for each key
  uint64_t full[C::kLoadChunks][C::kStages], empty[C::kLoadChunks][C::kStages];
  uint64_t scores[2], weights, done, queries, drained;
  uint32_t tmem;
  int32_t abort;
};
__device__ __forceinline__ int32_t ordered(float x) {
  const int32_t b = __float_as_int(x);
  return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float unordered(int32_t b) { return __int_as_float(b >= 0 ? b : b ^ 0x7fffffff); }

// A whole warp waits. A wait that ran out leaves *abort set, and every later
// wait returns at once: the loops then run to their end on whatever is there,
// so that each barrier gets the arrivals it counts, and the results are not
// stored.
__device__ __forceinline__ void warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  mbar_wait(smem_addr(bar), parity, abort);
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
    part[t] = lo | (static_cast<uint32_t>(hi) << 16);
    if (t + 1 < T) {
      const uint32_t a = wide ? e5m2x2_to_f16x2(lo) : e4m3x2_to_f16x2(lo);
      const uint32_t b = wide ? e5m2x2_to_f16x2(hi) : e4m3x2_to_f16x2(hi);
      const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
      const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
      r[0] -= fa.x;
      r[1] -= fa.y;
      r[2] -= fb.x;
      r[3] -= fb.y;
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
  part[0] = a1 | (static_cast<uint32_t>(b1) << 16);
  const uint16_t a2 = f16x2_to_e5m2x2(sub_f16x2(a, e4m3x2_to_f16x2(a1)));
  const uint16_t b2 = f16x2_to_e5m2x2(sub_f16x2(b, e4m3x2_to_f16x2(b1)));
  part[1] = a2 | (static_cast<uint32_t>(b2) << 16);
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

// A column of the CTA: which query (of the span) and head it is.
struct Column {
  int32_t query, head;
  bool used;
};

template <CacheShape SHAPE, int NH, int T>
__global__ void __launch_bounds__(Config<SHAPE, NH, T>::kThreads, Config<SHAPE, NH, T>::kPerSm)
    attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ AttendPlan plan) {
  using C = Config<SHAPE, NH, T>;
  using E = typename std::conditional<T == 2, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t smem[];
  using S = Shared<C, NH>;
  static_assert(C::kOffMisc + sizeof(S) <= C::kSmem, "shared state");
  S& sh = *reinterpret_cast<S*>(smem + C::kOffMisc);
  const uint32_t base = smem_addr(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(kAllLanes, tid >> 5, 0);
  constexpr int kMmaWarp = C::kThreads / 32 - 1;
  constexpr int kLoadWarp = C::kSoftmax / 32;

  // ---- set up, before the previous grid's results are needed
  if (tid == 0) {
    for (int c = 0; c < C::kLoadChunks; ++c) {
      for (int b = 0; b < C::kStages; ++b) {
        mbar_init(smem_addr(&sh.full[c][b]), C::kLoaders * (c == C::kNoteChunk ? 64 : 32));
        mbar_init(smem_addr(&sh.empty[c][b]), 1);
      }
    }
    mbar_init(smem_addr(&sh.scores[0]), 1);
    mbar_init(smem_addr(&sh.scores[1]), 1);
    mbar_init(smem_addr(&sh.weights), C::kSoftmax);
    mbar_init(smem_addr(&sh.done), 1);
    mbar_init(smem_addr(&sh.queries), C::kSoftmax);
    mbar_init(smem_addr(&sh.drained), 1);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (tid < NH) {
    sh.best[0][tid] = ordered(-INFINITY);
    sh.reference[tid] = 0.f;
  }
  if (warp == kMmaWarp) tmem_alloc(smem_addr(&sh.tmem), C::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(kAllLanes, sh.tmem, 0);
  volatile int* abort = &sh.abort;
  pdl_wait();
  pdl_launch_dependents();

  // ---- which work this CTA has
  const uint32_t ranks = cluster_size(), rank = cluster_ctarank();
  uint32_t unit = blockIdx.x / ranks;
  const int32_t block = unit % plan.blocks;
  unit /= plan.blocks;
  const int32_t kv = unit % a.cache.kv_heads;
  const int32_t item = unit / a.cache.kv_heads;
  QuerySpan span{item, 1, 0, 0};
  KeyList keys{};
  if (a.slots != nullptr) {
    keys = selected_keys(a, item);
  } else {
    span = find_span(a, item, plan.per);
    if (span.count > 0) keys = window_keys(a, span);
  }
  const int32_t tiles = (keys.n + kTile - 1) / kTile;
  const int32_t tile_begin = static_cast<int32_t>(static_cast<int64_t>(tiles) * rank / ranks);
  const int32_t tile_end = static_cast<int32_t>(static_cast<int64_t>(tiles) * (rank + 1) / ranks);
  const int32_t steps = tile_end - tile_begin;
  const bool several = span.count > 1;  // columns see different keys
  const int32_t group = a.heads_per_kv;
  auto column = [&](int32_t c) {
    Column r;
    r.query = plan.per.divisor == 1 ? 0 : c / group;
    const int32_t g = c - r.query * group + block * NH;
    r.head = kv * group + g;
    r.used = r.query < span.count && g < group && (plan.per.divisor == 1 || block == 0);
    return r;
  };

  if (tiles > 0) {
    if (warp < kLoadWarp) {
      // ================================================== queries, softmax
      const int wg = warp >> 2;
      const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // TMEM lane quadrant, << 16
      // -- split the queries: a warp takes four columns at a time, so that
      // their loads overlap
      constexpr int kPieces = (C::kKeyDim / 4 + 31) / 32;
      constexpr int kBatch = 4;
      for (int c0 = warp * kBatch; c0 < NH; c0 += kLoadWarp * kBatch) {
        uint2 raw[kBatch][kPieces];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const Column col = column(c0 + n);
          const E* q = static_cast<const E*>(a.q) + static_cast<int64_t>(span.row + col.query) * a.q_row +
                       static_cast<int64_t>(col.head) * a.q_head;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int d = (i * 32 + lane) * 4;
            raw[n][i] = make_uint2(0u, 0u);
            if (col.used && d < C::kKeyDim) raw[n][i] = *reinterpret_cast<const uint2*>(q + d);
          }
        }
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const int c = c0 + n;
          uint32_t most = 0;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            float x[4];
            unpack4<E>(raw[n][i], x);
#pragma unroll
            for (int k = 0; k < 4; ++k) most = max(most, __float_as_uint(x[k]) & 0x7fffffffu);
          }
          most = __reduce_max_sync(kAllLanes, most);
          // The largest magnitude comes to [128, 256): its exponent field is taken off.
          const int e = max(static_cast<int>(most >> 23), 40);
          const bool odd = most >= 0x7f800000u;  // an infinity or NaN: the row becomes NaN
          const float up = odd ? 0.f : __uint_as_float(static_cast<uint32_t>(134 + 127 - e) << 23);
          if (lane == 0) {
            sh.factor[c] = odd ? NAN : a.scale_log2 * __uint_as_float(static_cast<uint32_t>(e - 7) << 23);
            if constexpr (C::kSeveral) {
              const Column col = column(c);
              const int32_t position = span.position + col.query;
              sh.seen_to[c] = col.used ? position + 1 : 0x7fffffff;
              sh.seen_from[c] = col.used && a.window != 0 && position + 1 > static_cast<int64_t>(a.window)
                                    ? position + 1 - static_cast<int32_t>(a.window) : 0;
            }
          }
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int d = (i * 32 + lane) * 4;
            if (d < C::kKeyDim) {
              float y[4];
              unpack4<E>(raw[n][i], y);
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = odd ? 0.f : y[k] * up;
              uint32_t part[T];
              split4<T, false>(y, part);
              const int chunk = d / 128, in = d & 127;
              const bool narrow = C::kWide == 64 || (C::kIsLatent && chunk == 4);
#pragma unroll
              for (int t = 0; t < T; ++t) {
                const int row = t * NH + c;
                const uint32_t at = narrow ? row * 64 + ((((in >> 4) ^ (row >> 1)) & 3) << 4) + (in & 15)
                                           : row * 128 + ((((in >> 4) ^ row) & 7) << 4) + (in & 15);
                st_shared(base + C::kOffQ + chunk * (T * NH * 128) + at, part[t]);
              }
            }
          }
        }
      }
      fence_proxy_async();
      mbar_arrive(smem_addr(&sh.queries));
      named_barrier(1, C::kSoftmax);

      // -- tiles
      constexpr int CW = C::kCols;
      const int first_col = wg * CW;
      float l[CW];
#pragma unroll
      for (int c = 0; c < CW; ++c) l[c] = 0.f;
      float reference = -INFINITY, highest = -INFINITY;  // of column first_col + lane
      const int32_t all_to = span.position + 1;  // positions below are seen by every query, from
      const int32_t all_from =
          a.window == 0 ? 0
                        : static_cast<int32_t>(max(int64_t{0}, static_cast<int64_t>(span.position) + span.count - a.window));
      for (int32_t i = 0; i < steps; ++i) {
        warp_wait(&sh.scores[i & 1], (i >> 1) & 1, abort);
        tc_fence_after();
        const uint32_t b = i % C::kStages;
        warp_wait(&sh.full[C::kNoteChunk][b], (i / C::kStages) & 1, abort);
        const bool valid = (sh.valid[b][warp & 3] >> lane) & 1;
        const float ks = sh.k_scale[b][tid & 127];
        const float vs = C::kIsLatent ? ks : sh.v_scale[C::kIsLatent ? 0 : b][C::kIsLatent ? 0 : tid & 127];
        const uint32_t s_at = tmem + lanes + C::kValues * NH + (i & 1) * (T * NH) + first_col;
        float t[CW];
#pragma unroll
        for (int h = 0; h < CW; h += 16) {
          float s0[16], s1[16];
          tmem_ld16(s_at + h, s0);
          tmem_ld16(s_at + NH + h, s1);
          if constexpr (T == 3) {
            float s2[16];
            tmem_ld16(s_at + 2 * NH + h, s2);
            tmem_wait_ld(s0);
            tmem_wait_ld(s1);
            tmem_wait_ld(s2);
#pragma unroll
            for (int c = 0; c < 16; ++c) s1[c] += s2[c] * 0.0625f;
          } else {
            tmem_wait_ld(s0);
            tmem_wait_ld(s1);
          }
#pragma unroll
          for (int c = 0; c < 16; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(&sh.factor[first_col + h + c]);
            const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float s = (s0[c + k] + s1[c + k] * 0.0625f) * (ks * fs[k]);
              t[h + c + k] = valid ? s : -INFINITY;
            }
          }
        }
        if constexpr (C::kSeveral) {
          if (several) {
            const int32_t at = sh.position[b][tid & 127];
            const bool sink = static_cast<uint32_t>(at) < a.sinks;
            if (!(at < all_to && (at >= all_from || sink))) {
#pragma unroll
              for (int c = 0; c < CW; ++c) {
                const bool seen = at < sh.seen_to[first_col + c] && (at >= sh.seen_from[first_col + c] || sink);
                if (!seen) t[c] = -INFINITY;
              }
            }
          }
        }
        // Largest u of each column: lane c of a warp has column c's.
        const float scale = vs > 0.f ? fminf(fmaxf(vs, 0x1p-100f), 0x1p+100f) : vs;  // 0 and NaN stay
        const float shift = __log2f(scale > 0.f ? scale : 0x1p-100f);
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          const float m = warp_max(t[c] + shift);
          if ((lane & (CW - 1)) == c) top = m;
        }
        int32_t* best = sh.best[i % 3];
        if (lane < CW) {
          atomicMax(&best[first_col + lane], ordered(top));
          if ((warp & 3) == 0) sh.best[(i + 1) % 3][first_col + lane] = ordered(-INFINITY);
        }
        named_barrier(2 + wg, 128);
        top = unordered(best[first_col + (lane & (CW - 1))]);
        const bool move = top > reference + 3.5f || (top < reference - 4.f && top > highest - 60.f);
        bool waited = false;
        if (__any_sync(kAllLanes, move)) {
          const float to = move ? fmaxf(top, highest - 60.f) : reference;
          const float by = !move ? 1.f : reference == -INFINITY ? 0.f : exp2_approx(reference - to);
          reference = to;
          highest = fmaxf(highest, to);
          // The group's warps all write the same numbers: whoever reads them has
          // written them, and nobody is still at the tile before.
          if (lane < CW) sh.reference[first_col + lane] = to == -INFINITY ? 0.f : to;
          __syncwarp();
          if (i > 0) {
            warp_wait(&sh.done, (i - 1) & 1, abort);
            waited = true;
            tc_fence_after();
          }
#pragma unroll
          for (int h = 0; h < CW; h += 16) {
            float f[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              f[c] = __shfl_sync(kAllLanes, by, h + c);
              l[h + c] *= f[c];
            }
            if (i > 0) {
#pragma unroll 1
              for (int m = 0; m < C::kValues; ++m) {
                const uint32_t at = tmem + lanes + m * NH + first_col + h;
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
        }
        // Weights. The sum takes them in float32, the tensor core in T parts.
        const float to_value = scale * 32.f;
        uint32_t part[CW / 4][T];
#pragma unroll
        for (int c = 0; c < CW; c += 4) {
          const float4 r = *reinterpret_cast<const float4*>(&sh.reference[first_col + c]);
          const float rs[4] = {r.x, r.y, r.z, r.w};
          float w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float p = exp2_approx(t[c + k] - rs[k]);
            l[c + k] += p;
            w[k] = p * to_value;
          }
          if constexpr (T == 2) {
            split4_f16(w, part[c / 4]);
          } else {
            split4<T, true>(w, part[c / 4]);
          }
        }
        if (i > 0 && !waited) warp_wait(&sh.done, (i - 1) & 1, abort);
        const int row = tid & 127;
#pragma unroll
        for (int p = 0; p < T; ++p) {
#pragma unroll
          for (int h = 0; h < CW; h += 16) {
            const int piece = (first_col + h) / 16;
            const uint32_t at = NH == 64 ? row * 64 + ((piece ^ ((row >> 1) & 3)) << 4)
                                : NH == 32 ? row * 32 + ((piece ^ ((row >> 2) & 1)) << 4) : row * 16;
            st_shared_v4(base + C::kOffP + p * (NH * kTile) + at, part[h / 4][p], part[h / 4 + 1][p],
                         part[h / 4 + 2][p], part[h / 4 + 3][p]);
          }
        }
        fence_proxy_async();
        tc_fence_before();
        mbar_arrive(smem_addr(&sh.weights));
      }
      if (steps > 0) warp_wait(&sh.done, (steps - 1) & 1, abort);
      tc_fence_after();

      // -- sums over the keys: lanes first, then the group's warps. The
      // weights' buffer is free by now and takes the warps' sums.
      float* sums = reinterpret_cast<float*>(smem + C::kOffP) + wg * (4 * CW);
      float mine_l = sum_columns<CW>(l, lane);
      if (lane < CW) sums[(warp & 3) * CW + lane] = mine_l;
      named_barrier(2 + wg, 128);
      const int own = lane & (CW - 1);
      mine_l = (sums[own] + sums[CW + own]) + (sums[2 * CW + own] + sums[3 * CW + own]);

      float whole_l = mine_l, whole_r = reference, part_of = 1.f;
      if (ranks > 1) {
        // Every CTA's references and sums go round the cluster.
        float* joint = reinterpret_cast<float*>(smem + C::kOffP) + 8 * NH;  // references, then sums
        if ((warp & 3) == 0 && lane < CW) {
          joint[first_col + lane] = reference;
          joint[NH + first_col + lane] = mine_l;
        }
        cluster_sync();
        const uint32_t at = smem_addr(joint + first_col + own);
        whole_r = -INFINITY;
        for (uint32_t r = 0; r < ranks; ++r) whole_r = fmaxf(whole_r, ld_cluster(at, r));
        whole_l = 0.f;
        for (uint32_t r = 0; r < ranks; ++r) {
          const float rr = ld_cluster(at, r);
          whole_l += rr == -INFINITY ? 0.f : ld_cluster(at + NH * 4, r) * exp2_approx(rr - whole_r);
        }
        part_of = reference == -INFINITY ? 0.f : exp2_approx(reference - whole_r);
      }
      const float inverse = whole_l == 0.f ? 0.f : 1.f / (32.f * whole_l);
      if (rank == 0 && (warp & 3) == 0 && lane < CW && *abort == 0) {
        const Column col = column(first_col + lane);
        if (col.used) {
          a.lse[static_cast<int64_t>(span.row + col.query) * a.heads + col.head] =
              whole_l == 0.f ? -INFINITY : (whole_r + log2f(whole_l)) * 0.69314718055994531f;
        }
      }
      __syncwarp();
      if (lane < CW) sh.reference[first_col + lane] = part_of * inverse;
      __syncwarp();

      // -- outputs by way of the tiles' shared memory: in float32 to be joined
      // by the cluster, else as they are stored, in rows of a column
      constexpr int kRowsOf = SHAPE == kDim64 ? 64 : 128;  // of M = 128
      const bool failed = __any_sync(kAllLanes, *abort != 0);
      if (steps > 0 && !failed && (warp & 3) * 32 < kRowsOf) {
#pragma unroll 1
        for (int m = 0; m < C::kValues; ++m) {
          const int d = m * 128 + (warp & 3) * 32 + lane;
#pragma unroll
          for (int h = 0; h < CW; h += 16) {
            float o[16];
            tmem_ld16(tmem + lanes + m * NH + first_col + h, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const int at = (first_col + h + c) * C::kValueDim + d;
              const float y = o[c] * sh.reference[first_col + h + c];
              if (ranks > 1) {
                reinterpret_cast<float*>(smem)[at] = y;
              } else {
                reinterpret_cast<E*>(smem)[at] = static_cast<E>(y);
              }
            }
          }
        }
      }
      if (ranks == 1) {
        named_barrier(1, C::kSoftmax);
        if (!failed) {
          for (int c = warp; c < NH; c += kLoadWarp) {
            const Column col = column(c);
            if (!col.used) continue;
            E* out = static_cast<E*>(a.out) + static_cast<int64_t>(span.row + col.query) * a.out_row +
                     static_cast<int64_t>(col.head) * a.out_head;
            const E* from = reinterpret_cast<const E*>(smem) + c * C::kValueDim;
            if (a.out_wide) {
#pragma unroll
              for (int d = 0; d < C::kValueDim; d += 256) {
                if (d + lane * 8 < C::kValueDim) {
                  *reinterpret_cast<uint4*>(out + d + lane * 8) = *reinterpret_cast<const uint4*>(from + d + lane * 8);
                }
              }
            } else {
              for (int d = lane; d < C::kValueDim; d += 32) out[d] = from[d];
            }
          }
        }
      }
      tc_fence_before();
    } else if (warp < kMmaWarp) {
      // ================================================== gathering
      // A warp gathers its share of a tile's 128 rows; lane r knows the places
      // of rows r, r + 32, ..., eight lanes copy a 128-byte row (four a
      // 64-byte one).
      constexpr int kShare = kTile / C::kLoaders;   // rows of a warp
      constexpr int kOwn = kShare / 32;             // rows whose place a lane knows
      constexpr int kLanes = C::kWide / 16;         // lanes to a main row
      constexpr int kRows = 32 / kLanes;            // rows at once
      constexpr int kTurns = 32 / kRows;            // turns for 32 rows
      const int w = warp - kLoadWarp;
      const int32_t mine = tile_begin * kTile + w * kShare + lane;
      const uint8_t* k_base = a.cache.k + kv * a.cache.k_head;
      const uint8_t* v_base = a.cache.v + kv * a.cache.v_head;
      int32_t fetched[kOwn];
#pragma unroll
      for (int o = 0; o < kOwn; ++o) fetched[o] = steps > 0 ? fetch_key(a, keys, mine + o * 32) : -1;
      bool bad = false;
      uint32_t b = 0, turn = 0;
      for (int32_t i = 0; i < steps; ++i) {
        Key key[kOwn];
        uint32_t valid[kOwn];
        int64_t k_off[kOwn], v_off[kOwn];
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
          const int32_t j = mine + i * kTile + o * 32;
          key[o] = locate_key(a, keys, j, fetched[o]);
          bad |= bad_key(keys, j, fetched[o], key[o]);
          fetched[o] = i + 1 < steps ? fetch_key(a, keys, j + kTile) : -1;
          valid[o] = __ballot_sync(kAllLanes, key[o].valid);
          k_off[o] = key[o].block * a.cache.k_block + key[o].offset * a.cache.k_token;
          v_off[o] = key[o].block * a.cache.v_block + key[o].offset * a.cache.v_token;
        }
        // What the softmax has to know of a key: copied with its tile.
        auto note = [&]() {
#pragma unroll
          for (int o = 0; o < kOwn; ++o) {
            const int row = w * kShare + o * 32 + lane;
            const int64_t scale_at = static_cast<int64_t>(key[o].block) * a.cache.kv_heads + kv;
            cp_async4(smem_addr(&sh.k_scale[b][row]), a.cache.k_scale + scale_at, key[o].valid ? 4 : 0);
            if constexpr (!C::kIsLatent) {
              cp_async4(smem_addr(&sh.v_scale[b][row]), a.cache.v_scale + scale_at, key[o].valid ? 4 : 0);
            }
            if constexpr (C::kSeveral) sh.position[b][row] = key[o].position;
            if (lane == 0) sh.valid[b][w * kOwn + o] = valid[o];
          }
        };
        const uint32_t stage = base + b * C::kStageBytes;
        if constexpr (C::kIsLatent) {
          const uint8_t* from[kTurns];
#pragma unroll
          for (int n = 0; n < kTurns; ++n) {
            from[n] = k_base + __shfl_sync(kAllLanes, k_off[0], n * kRows + lane / kLanes) + (lane % kLanes) * 16;
          }
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            warp_wait(&sh.empty[c][b], turn ^ 1, abort);
#pragma unroll
            for (int n = 0; n < kTurns; ++n) {
              const int r = n * kRows + lane / kLanes, row = w * kShare + r;
              const uint32_t dst = stage + c * C::kChunkBytes + row * 128 + (((lane % 8) ^ (row & 7)) << 4);
              cp_async16(dst, from[n] + c * 128, (valid[0] >> r) & 1 ? 16 : 0);
            }
            if (c == C::kNoteChunk) {
              note();
              mbar_arrive(smem_addr(&sh.full[c][b]));
            }
            cp_async_arrive(smem_addr(&sh.full[c][b]));
          }
          const uint32_t tb = C::kTails == 1 ? 0 : b, tt = C::kTails == 1 ? i & 1 : turn;
          warp_wait(&sh.empty[4][tb], tt ^ 1, abort);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int r = n * 8 + lane / 4, row = w * kShare + r;
            const uint8_t* src = k_base + __shfl_sync(kAllLanes, k_off[0], r) + 512 + (lane % 4) * 16;
            const uint32_t dst = base + C::kOffTail + tb * C::kTailBytes + row * 64 + (((lane ^ (row >> 1)) & 3) << 4);
            cp_async16(dst, src, (valid[0] >> r) & 1 ? 16 : 0);
          }
          cp_async_arrive(smem_addr(&sh.full[4][tb]));
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            warp_wait(&sh.empty[c][b], turn ^ 1, abort);
            // 64-byte rows: values first, so that their second half of M reads
            // the keys behind them.
            const uint32_t at = stage + ((SHAPE == kDim64) == (c == 0) ? C::kChunkBytes : 0);
#pragma unroll
            for (int o = 0; o < kOwn; ++o) {
#pragma unroll
              for (int n = 0; n < kTurns; ++n) {
                const int r = n * kRows + lane / kLanes, row = w * kShare + o * 32 + r;
                const int64_t off = __shfl_sync(kAllLanes, c == 0 ? k_off[o] : v_off[o], r) + (lane % kLanes) * 16;
                const uint32_t dst = at + row * C::kWide + (C::kWide == 128 ? ((lane ^ row) & 7) << 4
                                                                            : ((lane ^ (row >> 1)) & 3) << 4);
                cp_async16(dst, (c == 0 ? k_base : v_base) + off, (valid[o] >> r) & 1 ? 16 : 0);
              }
            }
            if (c == C::kNoteChunk) {
              note();
              mbar_arrive(smem_addr(&sh.full[c][b]));
            }
            cp_async_arrive(smem_addr(&sh.full[c][b]));
          }
        }
        if (++b == C::kStages) {
          b = 0;
          turn ^= 1;
        }
      }
      cp_async_wait_all();
      if (__any_sync(kAllLanes, bad) && lane == 0) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
      if (ranks > 1) cluster_sync();
    } else {
      // ================================================== MMAs
      // The whole warp walks the loop, so that addresses stay in uniform
      // registers; one lane issues.
      if (steps > 0) {
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
        warp_wait(&sh.queries, 0, abort);
        uint32_t sb = 0, st = 0, ob = 0, ot = 0;  // stage and its turn, of scores and of outputs
        for (int32_t i = 0; i <= steps; ++i) {
          if (i < steps) {  // scores of tile i
            const uint32_t d = tmem + C::kValues * NH + (i & 1) * (T * NH);
#pragma unroll
            for (int c = 0; c < C::kMainKeys; ++c) {
              warp_wait(&sh.full[c][sb], st, abort);
              fence_proxy_async();
              if (leader) {
                const uint64_t kd = k_desc + ((sb * C::kStageBytes + c * C::kChunkBytes) >> 4);
                const uint64_t qd = q_desc + ((c * (T * NH * C::kWide)) >> 4);
#pragma unroll
                for (int k = 0; k < C::kWide / 32; ++k) mma_f8(d, kd + 2 * k, qd + 2 * k, kScoreDesc, c + k > 0);
              }
              __syncwarp();
            }
            if constexpr (C::kIsLatent) {
              const uint32_t tb = C::kTails == 1 ? 0 : sb, tt = C::kTails == 1 ? i & 1 : st;
              warp_wait(&sh.full[4][tb], tt, abort);
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
            if (leader) mma_commit(smem_addr(&sh.scores[i & 1]));
            __syncwarp();
            if (++sb == C::kStages) {
              sb = 0;
              st ^= 1;
            }
          }
          if (i > 0) {  // outputs of tile i - 1
            warp_wait(&sh.weights, (i - 1) & 1, abort);
            tc_fence_after();
            if constexpr (!C::kIsLatent) {
              warp_wait(&sh.full[1][ob], ot, abort);
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
                           p == 0 ? kFirstDesc : kOtherDesc, p + k > 0 || i > 1);
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
          }
        }
        if (__any_sync(kAllLanes, *abort != 0)) {  // gave up: let what was issued finish before the memory goes
          if (leader) {
            mma_commit(smem_addr(&sh.drained));
            const long long begin = clock64();
            while (!mbar_try(smem_addr(&sh.drained), 0) && clock64() - begin < 1000000000LL) {
            }
            flag_status(a.status, SILKERN_STATUS_WAIT_TIMEOUT);
          }
          __syncwarp();
        }
      }
      if (ranks > 1) cluster_sync();
    }

    if (ranks > 1) {
      // ==================================================== joining
      cluster_sync();
      const float* joint = reinterpret_cast<const float*>(smem + C::kOffP) + 8 * NH;
      for (int32_t e = (static_cast<int32_t>(rank) * C::kThreads + tid) * 4; e < NH * C::kValueDim;
           e += static_cast<int32_t>(ranks) * C::kThreads * 4) {
        const int32_t c = e / C::kValueDim, d = e - c * C::kValueDim;
        const Column col = column(c);
        if (!col.used) continue;
        float4 y{0.f, 0.f, 0.f, 0.f};
        for (uint32_t r = 0; r < ranks; ++r) {
          if (ld_cluster(smem_addr(joint + c), r) == -INFINITY) continue;  // rank r saw nothing
          const float4 x = ld_cluster4(base + e * 4, r);
          y.x += x.x;
          y.y += x.y;
          y.z += x.z;
          y.w += x.w;
        }
        E* out = static_cast<E*>(a.out) + static_cast<int64_t>(span.row + col.query) * a.out_row +
                 static_cast<int64_t>(col.head) * a.out_head + d;
        if (*abort == 0) {
          out[0] = static_cast<E>(y.x);
          out[1] = static_cast<E>(y.y);
          out[2] = static_cast<E>(y.z);
          out[3] = static_cast<E>(y.w);
        }
      }
      cluster_sync();  // nobody's shared memory goes before it was read
    }
  } else if (rank == 0) {
    // Nothing to see: out 0, lse -inf.
    for (int c = warp; c < NH; c += C::kThreads / 32) {
      const Column col = column(c);
      if (!col.used) continue;
      const int64_t row = span.row + col.query;
      E* out = static_cast<E*>(a.out) + row * a.out_row + static_cast<int64_t>(col.head) * a.out_head;
      for (int d = lane; d < C::kValueDim; d += 32) out[d] = static_cast<E>(0.f);
      if (lane == 0) a.lse[row * a.heads + col.head] = -INFINITY;
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, C::kColumns);
  }
}

template <CacheShape SHAPE, int NH, int T>
int launch_config(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  using C = Config<SHAPE, NH, T>;
  const int rc = allow_launch(reinterpret_cast<const void*>(attend_kernel<SHAPE, NH, T>), C::kSmem);
  if (rc != SILKERN_OK) return rc;
  return launch_pdl(attend_kernel<SHAPE, NH, T>, l.grid, C::kThreads, C::kSmem, l.cluster, l.stream, a, plan);
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
