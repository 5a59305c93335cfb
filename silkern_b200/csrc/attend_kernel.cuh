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
  static constexpr int kThreads = kSoftmax + 128 + 32;
  static constexpr int kQBytes = T * NH * kKeyDim;
  static constexpr int kPBytes = T * NH * kTile;
  static constexpr int kMisc = 3072;
  static constexpr int kColumnsUsed = kValues * NH + 2 * T * NH;
  static constexpr int kColumns = kColumnsUsed <= 128 ? 128 : kColumnsUsed <= 256 ? 256 : 512;
  static_assert(kColumnsUsed <= 512, "TMEM");
  // Two CTAs to an SM where a column block is narrow: each hides the other's
  // start, end and softmax. Otherwise one, with all of shared memory.
  static constexpr int kPerSm = !kIsLatent && NH == 16 ? 2 : 1;
  static constexpr int kSmemMax = smem_for_columns(512 / kPerSm);
  static constexpr int kFixed = kQBytes + kPBytes + kMisc;
  static constexpr int kStages = kIsLatent ? 2 : (kSmemMax - kFixed) / kStageBytes < 8 ? (kSmemMax - kFixed) / kStageBytes : 8;
  static constexpr int kTails = kIsLatent ? ((kSmemMax - kFixed - 2 * kStageBytes) >= 2 * kTailBytes ? 2 : 1) : 0;
  static constexpr int kUsed = kFixed + kStages * kStageBytes + kTails * kTailBytes;
  static_assert(kStages >= 2 && kUsed <= kSmemMax, "shared memory");
  static constexpr int kSmem = kUsed > smem_for_columns(kColumns) ? kUsed : smem_for_columns(kColumns);
  static_assert(NH * kValueDim * 4 <= kStages * kStageBytes, "joining buffer");
  // Offsets from the dynamic shared memory's start.
  static constexpr int kOffTail = kStages * kStageBytes;
  static constexpr int kOffQ = kOffTail + kTails * kTailBytes;
  static constexpr int kOffP = kOffQ + kQBytes;
  static constexpr int kOffMisc = kOffP + kPBytes;
};

// The small shared state behind the tiles.
template <int NH, int CHUNKS, int STAGES>
struct __align__(16) Shared {
  int32_t best[3][NH];     // running column maxima of a tile, as ordered integers
  float reference[8][32];  // each softmax warp's copy of its columns' references
  float factor[NH];        // score factor of a column, then 1 / (32 l)
  int32_t seen_to[NH], seen_from[NH];  // positions that a column sees: below, from
  uint64_t full[CHUNKS][STAGES], empty[CHUNKS][STAGES];
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
__device__ __forceinline__ void load4(const E* p, float (&x)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
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
  using S = Shared<NH, C::kLoadChunks, C::kStages>;
  static_assert(sizeof(S) <= C::kMisc, "shared state");
  S& sh = *reinterpret_cast<S*>(smem + C::kOffMisc);
  const uint32_t base = smem_addr(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kMmaWarp = C::kThreads / 32 - 1;
  constexpr int kLoadWarp = C::kSoftmax / 32;

  // ---- set up, before the previous grid's results are needed
  if (tid == 0) {
    for (int c = 0; c < C::kLoadChunks; ++c) {
      for (int b = 0; b < C::kStages; ++b) {
        mbar_init(smem_addr(&sh.full[c][b]), 128);
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
  if (tid < NH) sh.best[0][tid] = ordered(-INFINITY);
  if (warp == kMmaWarp) tmem_alloc(smem_addr(&sh.tmem), C::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
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
      // -- split the queries: a warp takes a column at a time
      for (int c = warp; c < NH; c += kLoadWarp) {
        const Column col = column(c);
        constexpr int kPieces = (C::kKeyDim / 4 + 31) / 32;
        float x[kPieces][4];
        uint32_t most = 0;
        const E* q = static_cast<const E*>(a.q) + static_cast<int64_t>(span.row + col.query) * a.q_row +
                     static_cast<int64_t>(col.head) * a.q_head;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int d = (i * 32 + lane) * 4;
          x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
          if (col.used && d < C::kKeyDim) load4(q + d, x[i]);
#pragma unroll
          for (int k = 0; k < 4; ++k) most = max(most, __float_as_uint(x[i][k]) & 0x7fffffffu);
        }
        most = __reduce_max_sync(kAllLanes, most);
        // The largest magnitude comes to [128, 256): its exponent field is taken off.
        const int e = max(static_cast<int>(most >> 23), 40);
        const bool odd = most >= 0x7f800000u;  // an infinity or NaN: the row becomes NaN
        const float up = odd ? 1.f : __uint_as_float(static_cast<uint32_t>(134 + 127 - e) << 23);
        if (lane == 0) {
          sh.factor[c] = odd ? NAN : a.scale_log2 * __uint_as_float(static_cast<uint32_t>(e - 7) << 23);
          const int32_t position = span.position + col.query;
          sh.seen_to[c] = col.used ? position + 1 : 0x7fffffff;
          sh.seen_from[c] = col.used && a.window != 0 && position + 1 > static_cast<int64_t>(a.window)
                                ? position + 1 - static_cast<int32_t>(a.window) : 0;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int d = (i * 32 + lane) * 4;
          if (d < C::kKeyDim) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = odd ? 0.f : x[i][k] * up;
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
      const int32_t mine = tile_begin * kTile + (tid & 127);
      const int32_t all_to = span.position + 1;  // positions below are seen by every query, from
      const int32_t all_from =
          a.window == 0 ? 0
                        : static_cast<int32_t>(max(int64_t{0}, static_cast<int64_t>(span.position) + span.count - a.window));
      int32_t fetched = fetch_key(a, keys, mine);
      Key key = locate_key(a, keys, mine, fetched);
      const int64_t kv_heads = a.cache.kv_heads;
      float ks = 0.f, vs = 0.f;
      if (key.valid) {
        ks = __ldg(a.cache.k_scale + key.block * kv_heads + kv);
        vs = C::kIsLatent ? ks : __ldg(a.cache.v_scale + key.block * kv_heads + kv);
      }
      fetched = fetch_key(a, keys, mine + kTile);
      if (lane < CW) sh.reference[warp][lane] = 0.f;
      __syncwarp();
      for (int32_t i = 0; i < steps; ++i) {
        // The next tile's key and scales, a tile ahead.
        const int32_t next_j = mine + (i + 1) * kTile;
        const Key next = i + 1 < steps ? locate_key(a, keys, next_j, fetched) : Key{0u, 0u, 0, false};
        float next_ks = 0.f, next_vs = 0.f;
        if (next.valid) {
          next_ks = __ldg(a.cache.k_scale + next.block * kv_heads + kv);
          next_vs = C::kIsLatent ? next_ks : __ldg(a.cache.v_scale + next.block * kv_heads + kv);
        }
        fetched = i + 2 < steps ? fetch_key(a, keys, next_j + kTile) : -1;

        warp_wait(&sh.scores[i & 1], (i >> 1) & 1, abort);
        tc_fence_after();
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
              t[h + c + k] = key.valid ? s : -INFINITY;
            }
          }
        }
        if (several && !(key.position < all_to &&
                         (key.position >= all_from || static_cast<uint32_t>(key.position) < a.sinks))) {
          const bool sink = static_cast<uint32_t>(key.position) < a.sinks;
#pragma unroll
          for (int c = 0; c < CW; ++c) {
            const bool seen = key.position < sh.seen_to[first_col + c] &&
                              (key.position >= sh.seen_from[first_col + c] || sink);
            if (!seen) t[c] = -INFINITY;
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
          __syncwarp();
          if (lane < CW) sh.reference[warp][lane] = to == -INFINITY ? 0.f : to;
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
          const float4 r = *reinterpret_cast<const float4*>(&sh.reference[warp][c]);
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
        key = next;
        ks = next_ks;
        vs = next_vs;
      }
      if (steps > 0) warp_wait(&sh.done, (steps - 1) & 1, abort);
      tc_fence_after();

      // -- sums over the keys: lanes first, then the group's warps. The
      // weights' buffer is free by now and takes the warps' sums.
      float* sums = reinterpret_cast<float*>(smem + C::kOffP) + wg * (4 * CW);
      float mine_l = 0.f;
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        float x = l[c];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(kAllLanes, x, d);
        if ((lane & (CW - 1)) == c) mine_l = x;
      }
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
      if (lane < CW) sh.reference[warp][lane] = part_of * inverse;
      __syncwarp();

      // -- outputs: straight from TMEM, or by way of shared memory to be joined
      const int rows_of = SHAPE == kDim64 ? 64 : 128;
      if (steps > 0 && !__any_sync(kAllLanes, *abort != 0)) {
        float* joined = reinterpret_cast<float*>(smem);
#pragma unroll 1
        for (int m = 0; m < C::kValues; ++m) {
          const int d = m * 128 + (warp & 3) * 32 + lane;
          if ((warp & 3) * 32 < rows_of) {
#pragma unroll 1
            for (int h = 0; h < CW; h += 16) {
              float o[16];
              tmem_ld16(tmem + lanes + m * NH + first_col + h, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const float y = o[c] * sh.reference[warp][h + c];
                if (ranks > 1) {
                  joined[(first_col + h + c) * C::kValueDim + d] = y;
                } else {
                  const Column col = column(first_col + h + c);
                  if (col.used) {
                    E* out = static_cast<E*>(a.out) + static_cast<int64_t>(span.row + col.query) * a.out_row +
                             static_cast<int64_t>(col.head) * a.out_head;
                    out[d] = static_cast<E>(y);
                  }
                }
              }
            }
          }
        }
      }
      tc_fence_before();
    } else if (warp < kMmaWarp) {
      // ================================================== gathering
      // A warp gathers 32 of a tile's 128 rows; lane r knows row r's place,
      // eight lanes copy a 128-byte row (four a 64-byte one).
      const int w = warp - kLoadWarp;
      const int32_t mine = tile_begin * kTile + w * 32 + lane;
      int32_t fetched = steps > 0 ? fetch_key(a, keys, mine) : -1;
      bool bad = false;
      constexpr int kLanes = C::kWide / 16;         // lanes to a main row
      constexpr int kRows = 32 / kLanes;            // rows at once
      constexpr int kTurns = 32 / kRows;
      for (int32_t i = 0; i < steps; ++i) {
        const int32_t j = mine + i * kTile;
        const Key key = locate_key(a, keys, j, fetched);
        bad |= bad_key(keys, j, fetched, key);
        fetched = i + 1 < steps ? fetch_key(a, keys, j + kTile) : -1;
        const uint32_t valid = __ballot_sync(kAllLanes, key.valid);
        const int64_t k_off = key.block * a.cache.k_block + key.offset * a.cache.k_token;
        const int64_t v_off = key.block * a.cache.v_block + key.offset * a.cache.v_token;
        const uint8_t* k_base = a.cache.k + kv * a.cache.k_head;
        const uint8_t* v_base = a.cache.v + kv * a.cache.v_head;
        const uint32_t b = i % C::kStages, turn = (i / C::kStages) & 1;
        const uint32_t stage = base + b * C::kStageBytes;
        if constexpr (C::kIsLatent) {
          const uint8_t* from[kTurns];
#pragma unroll
          for (int n = 0; n < kTurns; ++n) {
            from[n] = k_base + __shfl_sync(kAllLanes, k_off, n * kRows + lane / kLanes) + (lane % kLanes) * 16;
          }
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            warp_wait(&sh.empty[c][b], turn ^ 1, abort);
#pragma unroll
            for (int n = 0; n < kTurns; ++n) {
              const int r = n * kRows + lane / kLanes, row = w * 32 + r;
              const uint32_t dst = stage + c * C::kChunkBytes + row * 128 + (((lane % 8) ^ (row & 7)) << 4);
              cp_async16(dst, from[n] + c * 128, (valid >> r) & 1 ? 16 : 0);
            }
            cp_async_arrive(smem_addr(&sh.full[c][b]));
          }
          const uint32_t tb = i % C::kTails, tt = (i / C::kTails) & 1;
          warp_wait(&sh.empty[4][tb], tt ^ 1, abort);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int r = n * 8 + lane / 4, row = w * 32 + r;
            const uint8_t* src = k_base + __shfl_sync(kAllLanes, k_off, r) + 512 + (lane % 4) * 16;
            const uint32_t dst = base + C::kOffTail + tb * C::kTailBytes + row * 64 + (((lane ^ (row >> 1)) & 3) << 4);
            cp_async16(dst, src, (valid >> r) & 1 ? 16 : 0);
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
            for (int n = 0; n < kTurns; ++n) {
              const int r = n * kRows + lane / kLanes, row = w * 32 + r;
              const int64_t off = __shfl_sync(kAllLanes, c == 0 ? k_off : v_off, r) + (lane % kLanes) * 16;
              const uint32_t dst = at + row * C::kWide + (C::kWide == 128 ? ((lane ^ row) & 7) << 4
                                                                          : ((lane ^ (row >> 1)) & 3) << 4);
              cp_async16(dst, (c == 0 ? k_base : v_base) + off, (valid >> r) & 1 ? 16 : 0);
            }
            cp_async_arrive(smem_addr(&sh.full[c][b]));
          }
        }
      }
      cp_async_wait_all();
      if (__any_sync(kAllLanes, bad) && lane == 0) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
      if (ranks > 1) cluster_sync();
    } else {
      // ================================================== MMAs
      if (lane == 0 && steps > 0) {
        constexpr uint32_t kScoreDesc = mma_descriptor(128, T * NH, kE4M3, false, false);
        constexpr Swizzle kPSwizzle = NH == 64 ? kSwizzle64 : NH == 32 ? kSwizzle32 : kSwizzleNone;
        constexpr Swizzle kMain = C::kWide == 128 ? kSwizzle128 : kSwizzle64;
        const uint32_t q_at = base + C::kOffQ, p_at = base + C::kOffP;
        bool ok = mbar_wait(smem_addr(&sh.queries), 0, abort);
        int32_t issued = 0;
        for (int32_t i = 0; ok && i <= steps; ++i) {
          if (i < steps) {  // scores of tile i
            const uint32_t b = i % C::kStages, turn = (i / C::kStages) & 1;
            const uint32_t d = tmem + C::kValues * NH + (i & 1) * (T * NH);
#pragma unroll 1
            for (int c = 0; ok && c < C::kMainKeys; ++c) {
              ok = mbar_wait(smem_addr(&sh.full[c][b]), turn, abort);
              if (!ok) break;
              fence_proxy_async();
              const uint32_t k_at = base + b * C::kStageBytes + c * C::kChunkBytes + (SHAPE == kDim64 ? C::kChunkBytes : 0);
              const uint32_t qc = q_at + c * (T * NH * C::kWide);
#pragma unroll
              for (int k = 0; k < C::kWide / 32; ++k) {
                mma_f8(d, smem_descriptor(k_at + k * 32, 16, 8 * C::kWide, kMain),
                       smem_descriptor(qc + k * 32, 16, 8 * C::kWide, kMain), kScoreDesc, c + k > 0);
              }
            }
            if (!ok) break;
            if constexpr (C::kIsLatent) {
              const uint32_t tb = i % C::kTails;
              ok = mbar_wait(smem_addr(&sh.full[4][tb]), (i / C::kTails) & 1, abort);
              if (!ok) break;
              fence_proxy_async();
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                mma_f8(d, smem_descriptor(base + C::kOffTail + tb * C::kTailBytes + k * 32, 16, 512, kSwizzle64),
                       smem_descriptor(q_at + 4 * (T * NH * 128) + k * 32, 16, 512, kSwizzle64), kScoreDesc, true);
              }
              mma_commit(smem_addr(&sh.empty[4][tb]));
            } else {
              mma_commit(smem_addr(&sh.empty[0][b]));
            }
            mma_commit(smem_addr(&sh.scores[i & 1]));
          }
          if (i > 0) {  // outputs of tile i - 1
            const int32_t o = i - 1;
            const uint32_t b = o % C::kStages, turn = (o / C::kStages) & 1;
            ok = mbar_wait(smem_addr(&sh.weights), o & 1, abort);
            if (!ok) break;
            tc_fence_after();
            if constexpr (!C::kIsLatent) {
              ok = mbar_wait(smem_addr(&sh.full[1][b]), turn, abort);
              if (!ok) break;
              fence_proxy_async();
            }
#pragma unroll 1
            for (int c = 0; c < C::kValues; ++c) {
              const uint32_t v_at = base + b * C::kStageBytes + (SHAPE == kDim128 ? C::kChunkBytes : c * C::kChunkBytes);
#pragma unroll
              for (int p = 0; p < T; ++p) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  mma_f8(tmem + c * NH,
                         smem_descriptor(v_at + k * 32 * C::kWide, SHAPE == kDim64 ? C::kChunkBytes : 1024, 8 * C::kWide, kMain),
                         smem_descriptor(p_at + p * (NH * kTile) + k * 32 * NH, 8 * NH, 8 * NH, kPSwizzle),
                         p == 0 ? mma_descriptor(128, NH, kE4M3, true, true) : mma_descriptor(128, NH, kE5M2, true, true),
                         o + p + k > 0);
                }
              }
              mma_commit(smem_addr(&sh.empty[C::kIsLatent ? c : 1][b]));
            }
            mma_commit(smem_addr(&sh.done));
            issued = i;
          }
        }
        if (issued < steps) {  // gave up: let what was issued finish before the memory goes
          mma_commit(smem_addr(&sh.drained));
          const long long begin = clock64();
          while (!mbar_try(smem_addr(&sh.drained), 0) && clock64() - begin < 1000000000LL) {
          }
          flag_status(a.status, SILKERN_STATUS_WAIT_TIMEOUT);
        }
      }
      __syncwarp();
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
  const int rc = allow_shared_memory(reinterpret_cast<const void*>(attend_kernel<SHAPE, NH, T>), C::kSmem);
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
