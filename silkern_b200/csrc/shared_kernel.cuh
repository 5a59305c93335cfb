// Attention of a block of queries over a run of the 8-bit cache, on the
// fifth-generation tensor core.
//
//   S (128 rows x 128 keys) = Q K^T,   O (128 rows x dim) += P V
//
// A row is a (query, head) pair. A CTA has two slots of 128 rows, each with a
// softmax warpgroup, its scores and its outputs in TMEM; they share the K and V
// tiles where the block has more than 128 rows, and take turns with the tiles
// where it has less, so that one slot's softmax always runs beside the other's
// MMAs. Codes are widened to fp16, which holds e4m3 exactly, once for both slots:
// every multiply-add of the tensor core then is of 11-bit factors in float32.
//
// Q goes in as fp16 with a power of two for each row, its largest magnitude in
// [2^8, 2^9): exact but for columns below 2^-23 of the row's largest. The keys'
// scales, one for each page, are left to the scores: x = s kscale |softmax_scale|
// log2(e) 2^-row. Weights p = 2^(x - M) with M at most the largest x so far, and 8
// below it at most, so that O is rescaled seldom. What meets V is w = p vscale
// 2^(3 - E) in fp16, E the exponent of the first tile's largest value scale: with
// scales in [2^(E - 6), 2^(E + 4)) w is below 2^15, keeps 11 bits down to 2^-14 and
// half a step of 2^-25 below, 2^-28 of the largest weight. Tiles with other scales
// (and all after them) keep a reference R of their own for w = 2^(x + log2 vscale -
// R + 3), at a second exponential for each key and without the common case's
// straight code: 128 sequences of 64 heads behind 16384 tokens take 598 us instead of 190 where
// some CTAs meet such a tile early. Sums, M, R, S and O are float32.
//
// That w is one fp16 number is the price of one multiply-add for each key, where
// e4m3 and e5m2 parts would take two or three: 2^-11 of w at most where it is above
// 2^-14. Outputs' errors against 64 bits (relative, root mean square): bfloat16
// 1.675e-3 where float32 weights have 1.663e-3; float16 2.8e-4 and 3.0e-4 for 2.1e-4.
//
// A tile takes 3000 cycles with up to 128 rows, 3700 with up to 256; of these the
// tensor core 1300 and 2600, the exponentials 1024 and 2048. The first is bound by
// the latency of the codes' loads (a lane has registers for one tile of K and one
// of V on their way), the second by the chain of a half's scores, weights and
// outputs beside the other slot's. 128 sequences of 64 heads of 128 behind 32768
// shared tokens, with 20 to 1000 of their own: 238 us with plan and joining, 588
// TFLOP/s; 16 behind 131072: 137 us, 2.0 TB/s.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "host.cuh"
#include "ptx.cuh"
#include "shared_plan.cuh"
#include "silkern_b200.h"
#include "tcgen05.cuh"

namespace silkern {

namespace shared {

constexpr int kLoadWarps = 4;
constexpr int kMmaWarp = 8 + kLoadWarps;  // one for each slot
constexpr int kFenceWarp = kMmaWarp + 2;
constexpr int kWalkWarp = kFenceWarp + 1;
constexpr int kThreads = (kWalkWarp + 1) * 32;  // 512: up to 128 registers each
constexpr int kRing = 8;  // fragments known ahead
constexpr int kStages = 2;  // of K and of V
constexpr int kHalf = kSharedTile / 2;  // keys whose scores are there at once
constexpr int kNotes = 4;   // a tile's scales live until its V is read, three tiles of K later
// Weights go up to 2^kReach before their reference moves, and meet V times
// 2^kShift, with value scales in [2^(E - kBelow), 2^(E + kAbove + 1)): below 2^15.
constexpr int kReach = 8, kShift = 3, kAbove = 3, kBelow = 6;
static_assert(kReach + kShift + kAbove + 1 <= 15, "fp16 ends at 2^16");

struct __align__(16) Note {
  float k[kSharedTile];  // what a score is multiplied by
  float v[kSharedTile];  // value scales; -1: a key whose page is not in the cache
  // Largest and smallest exponent of value scales, whether such a key is among
  // them: of each loading warp's keys, and of the tile's.
  int4 seen[kLoadWarps], all;
};

// A part of an item and cache head that one CTA takes.
struct Fragment {
  int32_t kv;
  int32_t first, last;  // tiles; the CTA's last fragment is followed by one with last 0
  int32_t split;        // the slots take turns with the tiles
  int32_t lead;         // the slot that the first tile is then for
  int32_t key_begin, key_first, key_end;
  int32_t table_row;
  int32_t token, row, rows;
  int32_t seq, seqs;
  int32_t extra, prefix;
  int32_t one_half;     // the last tile has keys in its first half only

  // A slot's first tile, from the fragment's first on, and its half tiles.
  __device__ __forceinline__ int32_t own(int slot) const { return split ? slot ^ lead : 0; }
  __device__ __forceinline__ int32_t stride() const { return split ? 2 : 1; }
  __device__ __forceinline__ int32_t halves(int slot) const {
    const int32_t tiles = last - first, mine = split ? (tiles - own(slot) + 1) >> 1 : tiles;
    const bool has_last = !split || ((tiles - 1) & 1) == own(slot);
    return 2 * mine - (has_last ? one_half : 0);
  }
};

// A CTA's fragments, in order.
struct Walk {
  int64_t at, end;
  int32_t next_item, items;
  uint32_t tiles_before;
  SharedItem ahead;

  __device__ __forceinline__ void load_ahead(const SharedArgs& a) {
    if (next_item >= items) return;
    const int4* p = reinterpret_cast<const int4*>(a.item(next_item));
    int4* to = reinterpret_cast<int4*>(&ahead);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = __ldcg(p + i);
  }
  __device__ __forceinline__ void start(const SharedArgs& a) {
    const SharedHeader* h = a.header();
    const int64_t units = __ldcg(&h->units), share = __ldcg(&h->share);
    items = __ldcg(&h->items);
    at = share * blockIdx.x;
    end = min(at + share, units);
    next_item = 0;
    tiles_before = 0;
    if (at >= end) return;
    const int64_t heads = a.cache.kv_heads;
    next_item = warp_last_at_most(items, at, [&](int32_t i) { return __ldcg(&a.item(i)->begin) * heads; });
    load_ahead(a);
  }
  // The next fragment; false behind the last.
  __device__ __forceinline__ bool next(const SharedArgs& a, Fragment& f) {
    const int64_t heads = a.cache.kv_heads;
    while (at < end) {
      const int64_t cost = units_of(ahead.tiles, ahead.rows), base = ahead.begin * heads, inside = at - base;
      if (cost == 0 || inside >= cost * heads) {
        if (++next_item >= items) break;
        load_ahead(a);
        continue;
      }
      const int32_t each = units_of_tile(ahead.rows), kv = static_cast<int32_t>(inside / cost);
      const int64_t zero = base + kv * cost + units_of_start(ahead.rows);  // of the first tile
      auto tiles_before_unit = [&](int64_t unit) {
        return static_cast<int32_t>(unit <= zero ? 0 : min((unit - zero + each - 1) / each, static_cast<int64_t>(ahead.tiles)));
      };
      const int32_t first = tiles_before_unit(at), last = tiles_before_unit(end);
      f = Fragment{kv, first, last, ahead.rows <= kSlotRows ? 1 : 0, static_cast<int32_t>(tiles_before & 1),
                   ahead.key_begin, ahead.key_first, ahead.key_end, ahead.table_row, ahead.token, ahead.row, ahead.rows,
                   ahead.seq, ahead.seqs, ahead.extra, ahead.prefix,
                   ahead.key_end - ahead.key_begin - (last - 1) * kSharedTile <= kHalf ? 1 : 0};
      at = min(base + (kv + 1) * cost, end);
      if (kv + 1 == heads && at == base + heads * cost) {
        ++next_item;
        load_ahead(a);
      }
      if (last > first) {
        tiles_before += last - first;
        return true;
      }
    }
    return false;
  }
};

template <int DIM>
struct __align__(1024) Memory {
  uint8_t q[2][kSlotRows * DIM * 2];
  uint8_t k[kStages][kSharedTile * DIM * 2];
  uint8_t v[kStages][kSharedTile * DIM * 2];
  Note note[kNotes];
  Fragment ring[kRing];
  // [0]: of K, [1]: of V. Stored by the loading warps; ready for the MMAs; read by them.
  uint64_t stored[2][kStages], ready[2][kStages], free[2][kStages];
  uint64_t scores[2][2], weights[2][2], done[2][2];  // of a slot and half
  uint64_t queries[2], drained[2];
  uint64_t ring_full[kRing], ring_free[kRing];
  uint32_t tmem;
  int32_t abort;
};

// The piece of 16 bytes `piece` of row `row` of an operand tile: chunks of 64
// columns, 128 bytes a row, swizzled.
__device__ __forceinline__ uint32_t tile_place(uint32_t row, uint32_t piece) {
  return (piece >> 3) * (kSharedTile * 128) + row * 128 + (((piece ^ row) & 7) << 4);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
// A from TMEM: 128 lanes, two fp16 to a column.
__device__ __forceinline__ void mma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3])
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, float (&v)[8]) {  // and waits
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\ntcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
      : "r"(addr)
      : "memory");
}
using silkern::tmem_st16;
using silkern::tmem_wait_ld;
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]),
        "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]),
        "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
// The loaded registers may be used after this.
__device__ __forceinline__ void tmem_wait_ld(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
                 "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Half a tile's scores of one row, as its scales and masks make them: keys [low,
// high) count, and of them those whose page is in the cache.
struct Row {
  const float* k;  // of the half's keys
  const float* v;
  float unscale;
  int32_t low, high;
};

// All of these are short loops: an SM's warps run seven programs here, and straight
// code of some hundred instructions waits for its own fetching (64 keys unrolled
// took 1250 cycles, a masked half 15000).
//
// The usual half: nothing of it is hidden from the row, and each 16 keys share a
// page and its scales.
__device__ __forceinline__ float largest_plain(const Row& r, uint32_t s_at) {
  float most = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 32) {
    float x[32];
    tmem_ld32(s_at + c, x);
    const float k0 = r.k[c], k1 = r.k[c + 16];
    tmem_wait_ld(x);
    float b[4] = {x[0], x[1], x[16], x[17]};
#pragma unroll
    for (int i = 2; i < 14; i += 4) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        b[2 * j] = max3(b[2 * j], x[16 * j + i], x[16 * j + i + 1]);
        b[2 * j + 1] = max3(b[2 * j + 1], x[16 * j + i + 2], x[16 * j + i + 3]);
      }
    }
    most = max3(most, max3(b[0], b[1], fmaxf(x[14], x[15])) * k0, max3(b[2], b[3], fmaxf(x[30], x[31])) * k1);
  }
  return most * r.unscale;
}
// The weights against `base`: their sum is returned, their products with the value
// scales in `unit`s take the scores' place.
__device__ __forceinline__ float weigh_plain(const Row& r, uint32_t s_at, float base, float unit) {
  float sum0 = 0.f, sum1 = 0.f;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 16) {
    float x[16];
    uint32_t w[8];
    tmem_ld16(s_at + c, x);
    const float by = r.k[c] * r.unscale, vs = r.v[c] * unit;
    tmem_wait_ld(x);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float p0, p1, w0, w1;
      fma_pair(x[i], x[i + 1], by, by, -base, -base, p0, p1);
      p0 = exp2_approx(p0);
      p1 = exp2_approx(p1);
      add_pair(sum0, sum1, p0, p1, sum0, sum1);
      mul_pair(p0, p1, vs, vs, w0, w1);
      w[i / 2] = pack_f16x2(w0, w1);
    }
    tmem_st8(s_at + c / 2, w);
  }
  return sum0 + sum1;
}
// Both at once, against a reference that a score may turn out to pass (`best` says
// how far they went), so that the weights stay in registers: straight code, but
// the one that nearly every half takes.
__device__ __forceinline__ float weigh_ahead(const Row& r, uint32_t s_at, float base, float unit, float& best, uint32_t (&w)[2][16]) {
  float sum0 = 0.f, sum1 = 0.f, most = -INFINITY;
#pragma unroll
  for (int c = 0; c < kHalf; c += 32) {
    float x[32];
    tmem_ld32(s_at + c, x);
    tmem_wait_ld(x);
    float k[2], by[2], vs[2];
#pragma unroll
    for (int run = 0; run < 2; ++run) {
      k[run] = r.k[c + 16 * run];
      by[run] = k[run] * r.unscale;
      vs[run] = r.v[c + 16 * run] * unit;
      float b0 = x[16 * run], b1 = x[16 * run + 1];
#pragma unroll
      for (int i = 16 * run + 2; i < 16 * run + 16; i += 4) {
        b0 = max3(b0, x[i], x[i + 1]);
        if (i + 3 < 16 * run + 16) b1 = max3(b1, x[i + 2], x[i + 3]);
      }
      most = fmaxf(most, fmaxf(b0, b1) * k[run]);
    }
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const int run = i / 16;
      float p0, p1, w0, w1;
      fma_pair(x[i], x[i + 1], by[run], by[run], -base, -base, p0, p1);
      p0 = exp2_approx(p0);
      p1 = exp2_approx(p1);
      add_pair(sum0, sum1, p0, p1, sum0, sum1);
      mul_pair(p0, p1, vs[run], vs[run], w0, w1);
      w[c / 32][i / 2] = pack_f16x2(w0, w1);
    }
  }
  best = most * r.unscale;
  return sum0 + sum1;
}
// Any half: the largest score, and where value scales are far from the first tile's
// the largest of scores with log2 of their values' scales; then the weights.
__device__ __forceinline__ float score_of(const Row& r, int i, float x, float& vs) {
  vs = r.v[i];
  const float t = x * r.k[i] * r.unscale;
  return i >= r.low && i < r.high && !(vs < 0.f) ? t : -INFINITY;
}
__device__ __forceinline__ float largest_of_half(const Row& r, uint32_t s_at, bool usual, float& heaviest) {
  float best = -INFINITY;
  heaviest = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 8) {
    float x[8];
    tmem_ld8(s_at + c, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float vs;
      const float t = score_of(r, c + i, x[i], vs);
      best = fmaxf(best, t);
      if (!usual) heaviest = fmaxf(heaviest, t + __log2f(vs));
    }
  }
  return best;
}
__device__ __forceinline__ float weigh_half(const Row& r, uint32_t s_at, float base, float unit, bool usual, float reference) {
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 8) {
    float x[8];
    uint32_t w[4];
    tmem_ld8(s_at + c, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float vs;
      const float t = score_of(r, c + i, x[i], vs);
      const float p = exp2_approx(t - base);
      sum += p;
      x[i] = usual ? p * (vs * unit) : exp2_approx(t + __log2f(vs) - reference + kShift);
      if (t == -INFINITY) x[i] = 0.f;  // whatever its value's scale is
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_f16x2(x[2 * i], x[2 * i + 1]);
    tmem_st4(s_at + c / 2, w);
  }
  return sum;
}

template <typename T>
__device__ __forceinline__ float2 widen(uint32_t pair) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&pair));
  }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads, 1) shared_kernel(const __grid_constant__ SharedArgs a) {
  extern __shared__ __align__(1024) uint8_t raw_memory[];
  Memory<DIM>& m = *reinterpret_cast<Memory<DIM>*>(raw_memory);
  const int warp = __shfl_sync(kAllLanes, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kStages; ++i) {
      mbar_init(smem_addr(&m.stored[i / kStages][i % kStages]), kLoadWarps);
      mbar_init(smem_addr(&m.ready[i / kStages][i % kStages]), 1);
      mbar_init(smem_addr(&m.free[i / kStages][i % kStages]), 2);  // both slots' MMAs
    }
    for (int i = 0; i < 2; ++i) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_addr(&m.scores[i][h]), 1);
        mbar_init(smem_addr(&m.weights[i][h]), 4);
        mbar_init(smem_addr(&m.done[i][h]), 1);
      }
      mbar_init(smem_addr(&m.queries[i]), 4);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(smem_addr(&m.ring_full[i]), 1);
      mbar_init(smem_addr(&m.ring_free[i]), kWalkWarp);  // every other warp
    }
    mbar_init(smem_addr(&m.drained[0]), 1);
    mbar_init(smem_addr(&m.drained[1]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    m.abort = a.wait_cycles == 0 ? 1 : 0;
  }
  if (warp == kMmaWarp) tmem_alloc(smem_addr(&m.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(kAllLanes, m.tmem, 0);
  volatile int* abort = &m.abort;
  const int64_t bound = a.wait_cycles;
  pdl_wait();
  pdl_launch_dependents();
  constexpr uint32_t kScoresAt = 256;  // TMEM columns: outputs of the slots from 0 and DIM on, scores from here

  auto wait = [&](uint64_t* bar, uint32_t parity, int32_t tiles = 1) {  // a whole warp; false once a wait ran out
    return __all_sync(kAllLanes, mbar_wait(smem_addr(bar), parity, abort, bound * tiles)) != 0;
  };
  auto arrive = [&](uint64_t* bar) {  // once for the warp, behind all of its lanes
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(bar));
  };

  // The next fragment, behind `seq` others; false when there is none, or a wait ran
  // out. A warp that has read what it needs of it frees its place.
  auto next_fragment = [&](uint32_t seq) {
    return wait(&m.ring_full[seq % kRing], seq / kRing & 1) && m.ring[seq % kRing].last > 0;
  };
  auto free_fragment = [&](uint32_t seq) { arrive(&m.ring_free[seq % kRing]); };
  uint32_t seq = 0;

  if (warp < 8) {
    // ==================================================== softmax
    const int slot = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // TMEM lanes of this warp
    const uint32_t scores_at = tmem + lanes + kScoresAt + slot * kSharedTile, o_at = tmem + lanes + slot * DIM;
    const int row_in_slot = threadIdx.x & 127;
    uint32_t tiles_before = 0;  // of the CTA, for the notes' turns
    uint32_t parity = 0;  // bit h: of half h's scores
    bool going = true;
    for (; going && next_fragment(seq); ++seq) {
      const Fragment& f = m.ring[seq % kRing];
      const int32_t halves = f.halves(slot);
      const int32_t r = f.split ? row_in_slot : slot * kSlotRows + row_in_slot;  // this lane's, of the block
      const bool used = r < f.rows;
      const bool warp_used = __any_sync(kAllLanes, used);
      const int32_t row = f.row + (used ? r : 0), within = static_cast<int32_t>(fastdiv(row, a.per_kv));
      const int32_t token = f.token + within, head = f.kv * a.heads_per_kv + row - within * a.heads_per_kv;
      // Where its part of the result goes.
      int64_t place = static_cast<int64_t>(token) * a.heads + head;
      if (f.first > 0) {
        place = a.at.starts + blockIdx.x * static_cast<int64_t>(kBlockRows) + slot * kSlotRows + row_in_slot;
      } else if (f.split && slot == 1) {
        place = a.at.copies + static_cast<int64_t>(f.extra) * a.cache.kv_heads + static_cast<int64_t>(f.kv) * f.rows + r;
      } else if (f.prefix == 0) {
        place += static_cast<int64_t>(a.rows) * a.heads;
      }
      float result = -INFINITY, by_end = 0.f;  // log-sum-exp, factor of the outputs
      if (halves > 0) {
        // ---- the row's queries, in fp16, and how far it sees
        float unscale = 0.f;
        int32_t limit = 0;
        if (warp_used) {
          const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + token * a.q_row + head * a.q_head);
          uint4 x[DIM / 8];
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i) x[i] = __ldcg(q + i);
          const int32_t sequence = f.seqs == 1 ? f.seq : f.seq + last_at_most(f.seqs, token, [&](int32_t i) { return a.cu(f.seq + i); });
          const int64_t position = static_cast<int64_t>(load_int(a.lengths + sequence)) - (a.cu(sequence + 1) - token);
          limit = position < 0 ? 0 : a.keys_below(static_cast<int32_t>(position + 1));
          uint32_t most = 0;  // the largest magnitude, by its bits
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i) {
            most = __vmaxu2(most, __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                                           __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
          }
          most = max(most & 0xffffu, most >> 16);
          const float most_value = widen<T>(most).x;
          const int e = min(max(static_cast<int>(__float_as_uint(most_value) >> 23) - 127, -100), 127);
          unscale = __uint_as_float(static_cast<uint32_t>(e - 8 + 127) << 23);
          const float by = __uint_as_float(static_cast<uint32_t>(8 - e + 127) << 23) * a.q_sign;
          const uint32_t to = smem_addr(m.q[slot]);
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i) {
            const float2 b0 = widen<T>(x[i].x), b1 = widen<T>(x[i].y), b2 = widen<T>(x[i].z), b3 = widen<T>(x[i].w);
            st_shared_v4(to + tile_place(row_in_slot, i), pack_f16x2(b0.x * by, b0.y * by), pack_f16x2(b1.x * by, b1.y * by),
                         pack_f16x2(b2.x * by, b2.y * by), pack_f16x2(b3.x * by, b3.y * by));
          }
        }
        const int32_t all_see = __reduce_min_sync(kAllLanes, used ? min(limit, f.key_end) : 0x7fffffff);
        arrive(&m.queries[slot]);

        float top = -INFINITY, total = 0.f, reference = -INFINITY;
        int32_t exponent = 0;
        bool known = false, usual = true, pages = false;
        const int32_t stride = f.stride(), first_tile = f.own(slot);
        const int32_t key_first = f.key_first, seen = min(limit, f.key_end);
        int32_t first_key = f.key_begin + (f.first + first_tile) * kSharedTile;  // of the half
        const Note* note = nullptr;
        for (int32_t step = 0; step < halves; ++step) {
          const int half = step & 1;
          const uint32_t s_at = scores_at + half * kHalf;
          if (!wait(&m.scores[slot][half], parity >> half & 1)) {
            going = false;
            break;
          }
          parity ^= 1u << half;
          tc_fence_after();
          if (warp_used) {
            if (half == 0) {
              note = &m.note[(tiles_before + first_tile + (step >> 1) * stride) % kNotes];
              const int4 all = note->all;
              if (!known && all.x > -1000) {
                known = true;
                exponent = all.x;
              }
              if (usual && all.x > -1000 && (all.x > exponent + kAbove || all.y < exponent - kBelow)) {
                usual = false;
                reference = top + exponent;
              }
              pages = usual && a.runs && all.z == 0;
            }
            // Nothing of the half is hidden from any of the warp's rows.
            const bool plain = pages && key_first <= first_key && all_see - first_key >= kHalf;
            const Row at{note->k + half * kHalf, note->v + half * kHalf, unscale, key_first - first_key, seen - first_key};
            const float unit = __uint_as_float(static_cast<uint32_t>(127 + kShift - exponent) << 23);
            // ---- most halves leave the references where they are
            bool stays = plain && step > 0;
            if (stays) {
              uint32_t w[2][16];
              float best;
              const float sum = weigh_ahead(at, s_at, top == -INFINITY ? 0.f : top, unit, best, w);
              stays = __all_sync(kAllLanes, !(best > top + kReach));
              if (stays) {
                total += sum;
                tmem_st16(s_at, w[0]);
                tmem_st16(s_at + 16, w[1]);
              }
            }
            if (!stays) {
              float heaviest = -INFINITY;
              const float best = plain ? largest_plain(at, s_at) : largest_of_half(at, s_at, usual, heaviest);
              // References seldom move; then the sum and the outputs do.
              const bool up = best > top + kReach, heavier = heaviest > reference + kReach;
              if (__any_sync(kAllLanes, up || heavier)) {
                float by = 1.f;
                if (up) {
                  by = exp2f(top - best);
                  total *= by;
                  top = best;
                }
                if (!usual) {
                  by = heavier ? exp2f(reference - heaviest) : 1.f;
                  if (heavier) reference = heaviest;
                }
                if (step > 0) {
                  // The half before may still be added up.
                  if (!(going = wait(&m.done[slot][half ^ 1], (parity >> (half ^ 1) & 1) ^ 1))) break;
                  tc_fence_after();
  #pragma unroll 1
                  for (int c = 0; c < DIM; c += 16) {
                    float o[16];
                    tmem_ld16(o_at + c, o);
                    tmem_wait_ld(o);
  #pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] *= by;
                    tmem_st16(o_at + c, o);
                  }
                }
              }
              const float base = top == -INFINITY ? 0.f : top;
              total += plain ? weigh_plain(at, s_at, base, unit)
                             : weigh_half(at, s_at, base, unit, usual, reference == -INFINITY ? 0.f : reference);
            }
            tmem_wait_st();
          }
          tc_fence_before();
          arrive(&m.weights[slot][half]);
          first_key += half == 0 ? kHalf : stride * kSharedTile - kHalf;
        }
        if (!going) break;
        // 2^(reference - top - kShift) / total, in the usual case 2^(E - kShift) / total.
        const float lift = usual ? static_cast<float>(exponent) : reference - top;
        by_end = total > 0.f || total != total ? exp2f(lift - kShift) / total : 0.f;
        result = total == 0.f ? -INFINITY : top + log2f(total);
      }
      if (used) a.part_lse()[place] = result;
      if (halves > 0) {
        // (That the turns before the last are over follows from the last scores.)
        const int half = (halves - 1) & 1;
        if (!wait(&m.done[slot][half], (parity >> half & 1) ^ 1)) break;
        tc_fence_after();
        if (warp_used) {
          float4* out = reinterpret_cast<float4*>(a.part_out() + place * DIM);
#pragma unroll 1
          for (int c = 0; c < DIM; c += 32) {
            float o[32];
            tmem_ld32(o_at + c, o);
            tmem_wait_ld(o);
            if (used) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                out[c / 4 + i] = make_float4(o[4 * i] * by_end, o[4 * i + 1] * by_end, o[4 * i + 2] * by_end, o[4 * i + 3] * by_end);
              }
            }
          }
        }
        tc_fence_before();
      }
      tiles_before += f.last - f.first;
      free_fragment(seq);
    }
  } else if (warp < kMmaWarp) {
    // ==================================================== keys and values
    // A warp widens 32 of a tile's rows, 16 codes a lane at a time; each lane
    // knows the place of one. As soon as a tile's keys are stored the next
    // one's are on their way, and so the values: half a tile is in flight while
    // the other half is widened.
    constexpr int kLanes = DIM / 16;        // to a row
    constexpr int kAtOnce = 32 / kLanes;    // rows
    constexpr int kTurns = 32 / kAtOnce;
    const int w = warp - 8;
    const int known_row = kAtOnce * w + (lane & (kAtOnce - 1)) + kAtOnce * kLoadWarps * (lane / kAtOnce);
    // Eight neighbouring lanes take four pieces of two rows: with the swizzle,
    // their stores of 16 bytes reach all banks.
    const int my_row = kLanes == 4 ? lane >> 2 : (lane >> 2 & 1) | (lane >> 4 << 1);
    const int my_piece = kLanes == 4 ? lane & 3 : (lane & 3) | (lane >> 3 & 1) << 2;
    constexpr uint32_t kStep = kAtOnce * kLoadWarps * 128;  // from a row of this lane to the next: a multiple of 8 rows
    const uint32_t to = tile_place(kAtOnce * w + my_row, 2 * my_piece);
    bool bad = false;
    // The next tile, and the fragment that it belongs to.
    int32_t kv = 0, key = 0, key_first = 0, key_end = 0, tiles = 0, entry = 0;
    const int32_t* table = nullptr;
    auto advance = [&]() {  // to the next fragment; whether there is one
      if (!next_fragment(seq)) return false;
      const Fragment& f = m.ring[seq % kRing];
      kv = f.kv;
      key = f.key_begin + f.first * kSharedTile + known_row;  // this lane's
      key_first = f.key_first;
      key_end = f.key_end;
      tiles = f.last - f.first;
      table = a.table + f.table_row * static_cast<int64_t>(a.table_width);
      free_fragment(seq);
      ++seq;
      return true;
    };
    bool more = advance();
    // This lane's row of the next tile: its places, and its scales.
    int32_t k_row = -1, v_row = -1;
    float by = 0.f, vs = -1.f;
    bool counts = false;
    auto fetch = [&]() {  // the table's entry of the next tile
      entry = load_int(table + min(fastdiv(static_cast<uint32_t>(key), a.cache.block), a.table_width - 1));
    };
    auto locate = [&]() {  // places of the next tile, and the entry of the one behind it
      const uint32_t page = fastdiv(static_cast<uint32_t>(key), a.cache.block), block = static_cast<uint32_t>(entry);
      const uint32_t offset = key - page * a.cache.block.divisor;
      const bool wanted = key >= key_first && key < key_end;
      const bool held = page < a.table_width && block < a.cache.num_blocks;
      bad = bad || (wanted && !held);
      counts = wanted && held;
      k_row = counts ? static_cast<int32_t>(block * a.cache.k_block_rows + offset * a.cache.k_token_rows + kv * a.cache.k_head_rows) : -1;
      v_row = counts ? static_cast<int32_t>(block * a.cache.v_block_rows + offset * a.cache.v_token_rows + kv * a.cache.v_head_rows) : -1;
      by = 0.f;
      vs = wanted && !held ? -1.f : 0.f;
      if (held) {
        const int64_t s = static_cast<int64_t>(block) * a.cache.kv_heads + kv;
        by = __ldcg(a.cache.k_scale + s);
        vs = __ldcg(a.cache.v_scale + s);
      }
      key += kSharedTile;
      if (--tiles == 0) more = advance();
      if (more) fetch();
    };
    uint4 codes[2][kTurns];
    // (All exchanges come before the first load: they would wait for loads.)
    auto load = [&](uint4 (&c)[kTurns], const uint8_t* base, int64_t pitch, int32_t row) {
      int32_t r[kTurns];
#pragma unroll
      for (int i = 0; i < kTurns; ++i) r[i] = __shfl_sync(kAllLanes, row, my_row + kAtOnce * i);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        asm volatile(
            "{\n .reg .pred p;\n setp.ge.s32 p, %5, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n"
            " @p ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n}"
            : "=&r"(c[i].x), "=&r"(c[i].y), "=&r"(c[i].z), "=&r"(c[i].w)
            : "l"(base + r[i] * pitch + my_piece * 16), "r"(r[i])
            : "memory");
      }
    };
    auto widen_to = [&](uint32_t tile_at, const uint4 (&codes)[kTurns]) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const uint32_t c[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[2 * k] = e4m3x2_to_f16x2(static_cast<uint16_t>(c[k] & 0xffffu));
          h[2 * k + 1] = e4m3x2_to_f16x2(static_cast<uint16_t>(c[k] >> 16));
        }
        st_shared_v4(tile_at + to + i * kStep, h[0], h[1], h[2], h[3]);
        st_shared_v4(tile_at + (to ^ 16) + i * kStep, h[4], h[5], h[6], h[7]);
      }
    };
    // Keys are stored a tile ahead of the values: the slots take turns with the
    // tiles, and one's next scores must not wait for the other's weights.
    if (more) {
      fetch();
      locate();
      load(codes[0], a.cache.k, a.cache.k_pitch, k_row);
      load(codes[1], a.cache.v, a.cache.v_pitch, v_row);
      auto store_values = [&](uint32_t turn) {
        const uint32_t stage = turn % kStages;
        if (!wait(&m.free[1][stage], (turn / kStages & 1) ^ 1)) return false;
        widen_to(smem_addr(m.v[stage]), codes[1]);
        arrive(&m.stored[1][stage]);
        return true;
      };
      bool going = true;
      uint32_t turn = 0;
      for (bool ahead = true; ahead && going; ++turn) {
        const float tile_by = by * a.scale_log2, tile_vs = vs;
        const bool tile_counts = counts;
        const int32_t tile_v_row = v_row;
        ahead = more;
        if (ahead) locate();
        const uint32_t stage = turn % kStages;
        if (!wait(&m.free[0][stage], (turn / kStages & 1) ^ 1)) {
          going = false;
          break;
        }
        widen_to(smem_addr(m.k[stage]), codes[0]);
        Note& note = m.note[turn % kNotes];
        const int32_t e = static_cast<int32_t>(__float_as_uint(tile_vs) >> 23 & 0xff);
        const bool known = tile_counts && tile_vs > 0.f && e != 255;  // neither 0 nor NaN
        const int32_t most = __reduce_max_sync(kAllLanes, known ? e - 127 : -1000);
        const int32_t least = __reduce_min_sync(kAllLanes, known ? e - 127 : 1000);
        const bool holes = __any_sync(kAllLanes, tile_vs < 0.f);
        note.k[known_row] = tile_by;
        note.v[known_row] = tile_vs;
        if (lane == 0) note.seen[w] = make_int4(most, least, holes ? 1 : 0, 0);
        arrive(&m.stored[0][stage]);
        if (ahead) load(codes[0], a.cache.k, a.cache.k_pitch, k_row);
        if (turn > 0) {
          going = store_values(turn - 1);
          if (going) load(codes[1], a.cache.v, a.cache.v_pitch, tile_v_row);
        }
      }
      if (going) store_values(turn - 1);
    }
    if (bad) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
  } else if (warp < kFenceWarp) {
    // ==================================================== MMAs
    // A warp for each slot. All of it walks, so that descriptors stay in uniform
    // registers; one lane issues. Each passes every tile, its own or not, so that
    // their places fill in turn.
    constexpr uint32_t kScoreDesc = mma_descriptor(128, kHalf, 0, false, false);
    constexpr uint32_t kOutDesc = mma_descriptor(128, DIM, 0, false, true);
    constexpr uint32_t kChunk = kSharedTile * 128;  // bytes of 64 columns of a tile
    constexpr uint32_t kTileStep = kSharedTile * DIM * 2 >> 4, kHalfStep = kHalf * 128 >> 4;  // in units of 16 bytes
    const int slot = warp - kMmaWarp;
    const bool leader = elect_one();
    const uint64_t q_desc = smem_descriptor(smem_addr(m.q[slot]), 16, 1024, kSwizzle128);
    const uint64_t k_desc = smem_descriptor(smem_addr(m.k[0]), 16, 1024, kSwizzle128);
    const uint64_t v_desc = smem_descriptor(smem_addr(m.v[0]), kChunk, 1024, kSwizzle128);
    const uint32_t scores_at = tmem + kScoresAt + slot * kSharedTile, o_at = tmem + slot * DIM;
    uint32_t tiles_before = 0, k_next = 0, v_next = 0;  // tiles of the CTA: before the fragment, not waited for yet
    uint32_t queries_parity = 0, weights_parity = 0;    // (a bit for each half)
    bool going = true;
    // Up to `tile`, of K (0) or V (1): the others' tiles are passed, and it is there.
    auto reach = [&](int which, uint32_t& next, uint32_t tile) {
      for (; next <= tile; ++next) {
        if (!wait(&m.ready[which][next % kStages], next / kStages & 1)) return false;
        if (next < tile) arrive(&m.free[which][next % kStages]);
      }
      return true;
    };
    for (; going && next_fragment(seq); ++seq) {
      const Fragment& f = m.ring[seq % kRing];
      const int32_t tiles = f.last - f.first, halves = f.halves(slot);
      const uint32_t own = tiles_before + f.own(slot), stride = f.stride();
      free_fragment(seq);
      // Scores run two halves ahead of the outputs, so that the softmax finds the
      // next ones when it is through with a half.
      for (int32_t i = -2; i < halves; ++i) {
        const uint32_t half = i & 1, s_at = scores_at + half * kHalf;
        if (i >= 0) {  // outputs
          const uint32_t tile = own + (i >> 1) * stride, stage = tile % kStages;
          if (half == 0 && !(going = reach(1, v_next, tile))) break;
          if (!(going = wait(&m.weights[slot][half], weights_parity >> half & 1))) break;
          weights_parity ^= 1u << half;
          tc_fence_after();
          const uint64_t vd = v_desc + stage * kTileStep + half * kHalfStep;
          if (leader) {
#pragma unroll
            for (int k = 0; k < kHalf / 16; ++k) {
              mma_f16_tmem(o_at, s_at + k * 8, vd + (k * 2048 >> 4), kOutDesc, k > 0 || i > 0);
            }
            mma_commit(smem_addr(&m.done[slot][half]));
            if (half == 1 || i + 1 == halves) mma_commit(smem_addr(&m.free[1][stage]));
          }
          __syncwarp();
        }
        if (i + 2 < halves) {  // scores
          const uint32_t tile = own + ((i + 2) >> 1) * stride, stage = tile % kStages;
          if (half == 0 && !(going = reach(0, k_next, tile))) break;
          if (i == -2) {
            if (!(going = wait(&m.queries[slot], queries_parity))) break;
            queries_parity ^= 1;
            fence_proxy_async();  // (the softmax would wait for its stores to global memory)
            tc_fence_after();
          }
          const uint64_t kd = k_desc + stage * kTileStep + half * kHalfStep;
          if (leader) {
#pragma unroll
            for (int k = 0; k < DIM / 16; ++k) {
              const uint32_t at = (k / 4 * kChunk + k % 4 * 32) >> 4;
              mma_f16(s_at, q_desc + at, kd + at, kScoreDesc, k > 0);
            }
            mma_commit(smem_addr(&m.scores[slot][half]));
            if (half == 1 || i + 3 == halves) mma_commit(smem_addr(&m.free[0][stage]));
          }
          __syncwarp();
        }
      }
      tiles_before += tiles;
      // The other slot's last tile.
      if (going && k_next < tiles_before) {
        going = reach(0, k_next, tiles_before - 1);
        if (going) arrive(&m.free[0][(tiles_before - 1) % kStages]);
      }
      if (going && v_next < tiles_before) {
        going = reach(1, v_next, tiles_before - 1);
        if (going) arrive(&m.free[1][(tiles_before - 1) % kStages]);
      }
    }
    // However the walk ended, what this lane issued finishes before the memory and
    // the TMEM go: where another warp gave up, nothing else waits for it. (Elsewhere
    // the softmax waits as long.)
    if (leader) {
      mma_commit(smem_addr(&m.drained[slot]));
      const long long begin = clock64();
      while (!mbar_try(smem_addr(&m.drained[slot]), 0) && clock64() - begin < 4000000000LL) {
      }
    }
    __syncwarp();
  } else if (warp == kFenceWarp) {
    // ==================================================== from stores to operands
    // The loading warps store through the generic proxy, the tensor core reads
    // through another. The fence between takes hundreds of cycles, of a loading
    // warp until its loads are in, of an MMAs' warp while the tensor core waits.
    uint32_t turn = 0;
    bool going = true;
    auto pass = [&](int which, uint32_t tile) {
      const uint32_t stage = tile % kStages;
      if (!wait(&m.stored[which][stage], tile / kStages & 1)) return false;
      if (which == 0 && lane == 0) {
        Note& note = m.note[tile % kNotes];
        int4 all = note.seen[0];
#pragma unroll
        for (int k = 1; k < kLoadWarps; ++k) {
          all = make_int4(max(all.x, note.seen[k].x), min(all.y, note.seen[k].y), all.z | note.seen[k].z, 0);
        }
        note.all = all;
      }
      fence_proxy_async();
      arrive(&m.ready[which][stage]);
      return true;
    };
    for (; going && next_fragment(seq); ++seq) {
      const int32_t tiles = m.ring[seq % kRing].last - m.ring[seq % kRing].first;
      free_fragment(seq);
      for (int32_t i = 0; i < tiles && going; ++i, ++turn) {
        going = pass(0, turn) && (turn == 0 || pass(1, turn - 1));
      }
    }
    if (going && turn > 0) pass(1, turn - 1);
  } else {
    // ==================================================== the CTA's fragments
    Walk walk;
    Fragment f;
    walk.start(a);
    for (bool more = true; more; ++seq) {
      more = walk.next(a, f);
      if (!more) f.last = 0;
      // (The place's last fragment may have only begun.)
      Fragment& to = m.ring[seq % kRing];
      if (!wait(&m.ring_free[seq % kRing], (seq / kRing & 1) ^ 1, seq < kRing ? 1 : 2 + to.last - to.first)) break;
      __syncwarp();
      if (lane == 0) to = f;
      arrive(&m.ring_full[seq % kRing]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_free(tmem, 512);
  if (threadIdx.x == 0 && *abort != 0) {
    atomicExch(&a.header()->failed, 1);
    flag_status(a.status, SILKERN_STATUS_WAIT_TIMEOUT);
  }
}

template <typename T, int DIM>
int launch(const SharedArgs& a, unsigned grid, cudaStream_t stream) {
  static DeviceBits granted{0};
  constexpr int bytes = static_cast<int>(sizeof(Memory<DIM>));
  static_assert(bytes <= 227 * 1024, "shared memory");
  void (*fn)(SharedArgs) = shared_kernel<T, DIM>;
  const int rc = allow_launch(reinterpret_cast<const void*>(fn), bytes, granted);
  if (rc != SILKERN_OK) return rc;
  return launch_pdl(fn, grid, kThreads, bytes, 1, stream, a);
}

}  // namespace shared
}  // namespace silkern
