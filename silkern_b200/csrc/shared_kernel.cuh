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
// log2(e) 2^-row. Weights p = 2^(x - M) with M at most the largest x so far, and 4
// below it at most, so that O is rescaled seldom. What meets V is w = p vscale
// 2^(6 - E) in fp16, E the exponent of the first tile's largest value scale: with
// scales in [2^(E - 8), 2^(E + 4)) w is below 2^15, keeps 11 bits down to 2^-14 and
// half a step of 2^-25 below, 2^-31 of the largest weight. Tiles with other scales
// (and all after them) keep a reference R of their own for w = 2^(x + log2 vscale -
// R + 6), at a second exponential for each key. Sums, M, R, S and O are float32.
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

constexpr int kLoadWarps = 8;
constexpr int kMmaWarp = 8 + kLoadWarps;
constexpr int kThreads = (kMmaWarp + 1) * 32;
constexpr int kStages = 2;  // of K and of V
constexpr int kNotes = 3;   // a tile's scales live until its V is read

struct Note {
  float k[kSharedTile];  // what a score is multiplied by
  float v[kSharedTile];  // value scales; -1: a key that does not count
  int4 seen[kLoadWarps]; // largest and smallest exponent of value scales, whether a key does not count
};

template <int DIM>
struct __align__(1024) Memory {
  uint8_t q[2][kSlotRows * DIM * 2];
  uint8_t k[kStages][kSharedTile * DIM * 2];
  uint8_t v[kStages][kSharedTile * DIM * 2];
  Note note[kNotes];
  uint64_t k_full[kStages], k_free[kStages], v_full[kStages], v_free[kStages];
  uint64_t scores[2], weights[2], queries[2], done[2], drained;
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

// A part of an item and cache head that one CTA takes.
struct Fragment {
  SharedItem item;
  int32_t kv;
  int32_t first, last;  // tiles
  bool split;           // the slots take turns with the tiles

  // Tiles of a slot.
  __device__ __forceinline__ int32_t steps(int slot) const {
    return split ? (last - first + 1 - slot) >> 1 : last - first;
  }
  __device__ __forceinline__ int32_t tile(int slot, int32_t step) const {
    return first + (split ? 2 * step + slot : step);
  }
};

// A CTA's fragments, in order.
struct Walk {
  int64_t at, end;
  int32_t next_item, items;
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
    if (at >= end) return;
    const int64_t heads = a.cache.kv_heads;
    next_item = warp_last_at_most(items, at, [&](int32_t i) { return __ldcg(&a.item(i)->begin) * heads; });
    load_ahead(a);
  }
  // The next fragment; false behind the last.
  __device__ __forceinline__ bool next(const SharedArgs& a, Fragment& f) {
    const int64_t heads = a.cache.kv_heads;
    while (at < end) {
      const int32_t cost = units_of(ahead.tiles);
      const int64_t base = ahead.begin * heads;
      const int64_t inside = at - base;
      if (cost == 0 || inside >= cost * heads) {
        if (++next_item >= items) break;
        load_ahead(a);
        continue;
      }
      const int32_t kv = static_cast<int32_t>(inside / cost);
      const int64_t zero = base + static_cast<int64_t>(kv) * cost + kStart;  // of the first tile
      const int64_t last = min(end - zero, static_cast<int64_t>(ahead.tiles));
      const int64_t first = max(at - zero, int64_t{0});
      f.item = ahead;
      f.kv = kv;
      f.first = static_cast<int32_t>(first);
      f.last = static_cast<int32_t>(last);
      f.split = ahead.rows <= kSlotRows;
      at = min(zero + ahead.tiles, end);
      if (kv + 1 == heads && at == zero + ahead.tiles) {
        ++next_item;
        load_ahead(a);
      }
      if (last > first) return true;
    }
    return false;
  }
};

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
  extern __shared__ uint8_t raw_memory[];
  Memory<DIM>& m = *reinterpret_cast<Memory<DIM>*>((reinterpret_cast<uintptr_t>(raw_memory) + 1023) & ~uintptr_t{1023});
  const int warp = __shfl_sync(kAllLanes, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_addr(&m.k_full[i]), kLoadWarps);
      mbar_init(smem_addr(&m.v_full[i]), kLoadWarps);
      mbar_init(smem_addr(&m.k_free[i]), 1);
      mbar_init(smem_addr(&m.v_free[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&m.scores[i]), 1);
      mbar_init(smem_addr(&m.weights[i]), 4);
      mbar_init(smem_addr(&m.queries[i]), 4);
      mbar_init(smem_addr(&m.done[i]), 1);
    }
    mbar_init(smem_addr(&m.drained), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    m.abort = 0;
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

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    mbar_wait(smem_addr(bar), parity, abort, bound);
    return !__any_sync(kAllLanes, *abort != 0);
  };
  auto arrive = [&](uint64_t* bar) {  // once for the warp, behind all of its lanes
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(bar));
  };

  Walk walk;
  Fragment f;
  walk.start(a);

  if (warp < 8) {
    // ==================================================== softmax
    const int slot = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // TMEM lanes of this warp
    const uint32_t s_at = tmem + lanes + kScoresAt + slot * kSharedTile, o_at = tmem + lanes + slot * DIM;
    const int row_in_slot = threadIdx.x & 127;
    uint32_t tiles_before = 0;  // of the CTA, for the notes' turns
    uint32_t turn = 0, done_turn = 0;
    bool going = true;
    while (going && walk.next(a, f)) {
      const SharedItem& it = f.item;
      const int32_t steps = f.steps(slot);
      const int32_t r = f.split ? row_in_slot : slot * kSlotRows + row_in_slot;  // of the block
      const bool used = r < it.rows;
      const bool warp_used = __any_sync(kAllLanes, used);
      const int32_t row = it.row + (used ? r : 0);
      const int32_t within = static_cast<int32_t>(fastdiv(row, a.per_kv));
      const int32_t token = it.token + within;
      const int32_t head = f.kv * a.heads_per_kv + row - within * a.heads_per_kv;
      if (steps > 0) {
        // ---- the row's queries, and how far it sees
        float unscale = 0.f;
        int32_t limit = 0;
        if (warp_used) {
          const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + token * a.q_row + head * a.q_head);
          uint4 x[DIM / 8];
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i) x[i] = __ldcg(q + i);
          const int32_t seq = it.seqs == 1 ? it.seq : it.seq + last_at_most(it.seqs, token, [&](int32_t i) { return a.cu(it.seq + i); });
          const int64_t position = static_cast<int64_t>(load_int(a.lengths + seq)) - (a.cu(seq + 1) - token);
          limit = position < 0 ? 0 : a.keys_below(static_cast<int32_t>(position + 1));
          uint32_t most = 0;  // the largest magnitude, by its bits
#pragma unroll
          for (int i = 0; i < DIM / 8; ++i) {
            most = __vmaxu2(most, __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                                           __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
          }
          most = max(most & 0xffffu, most >> 16);
          const float largest = widen<T>(most).x;
          const int e = min(max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -100), 127);
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
        fence_proxy_async();
        arrive(&m.queries[slot]);

        float top = -INFINITY, total = 0.f, reference = -INFINITY;
        int32_t exponent = 0;
        bool known = false, usual = true;
        for (int32_t step = 0; step < steps; ++step) {
          const int32_t tile = f.tile(slot, step);
          const Note& note = m.note[(tiles_before + static_cast<uint32_t>(tile - f.first)) % kNotes];
          if (!wait(&m.scores[slot], turn & 1)) {
            going = false;
            break;
          }
          ++turn;
          tc_fence_after();
          if (warp_used) {
            int32_t most = -1000, least = 1000, holes = 0;
#pragma unroll
            for (int i = 0; i < kLoadWarps; ++i) {
              const int4 s = note.seen[i];
              most = max(most, s.x);
              least = min(least, s.y);
              holes |= s.z;
            }
            if (!known && most > -1000) {
              known = true;
              exponent = most;
            }
            if (usual && most > -1000 && (most > exponent + 3 || least < exponent - 8)) {
              usual = false;
              reference = top + exponent;
            }
            const int32_t first_key = it.key_begin + tile * kSharedTile;
            const bool masked = holes != 0 || __any_sync(kAllLanes, used && limit < first_key + kSharedTile);
            const int32_t seen = limit - first_key;  // keys of the tile that the row may see
            // ---- the largest score, and the largest weight where values' scales count
            float best = -INFINITY, heaviest = -INFINITY;
            if (usual && !masked && a.runs) {
#pragma unroll 1
              for (int c = 0; c < 8; c += 2) {
                float x[16], y[16];
                tmem_ld16(s_at + c * 16, x);
                tmem_ld16(s_at + c * 16 + 16, y);
                tmem_wait_ld(x);
                tmem_wait_ld(y);
                float b0 = x[0], b1 = y[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) {
                  b0 = fmaxf(b0, x[i]);
                  b1 = fmaxf(b1, y[i]);
                }
                best = fmaxf(best, fmaxf(b0 * note.k[c * 16], b1 * note.k[c * 16 + 16]));
              }
              best *= unscale;
            } else {
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {
                float x[16];
                tmem_ld16(s_at + c * 16, x);
                tmem_wait_ld(x);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float vs = note.v[c * 16 + i];
                  if (!(vs < 0.f) && c * 16 + i < seen) {
                    const float t = x[i] * note.k[c * 16 + i] * unscale;
                    best = fmaxf(best, t);
                    if (!usual) heaviest = fmaxf(heaviest, t + log2f(vs));
                  }
                }
              }
            }
            // ---- references move, with the sum and the outputs
            const bool up = best > top + 4.f || (top == -INFINITY && best > top);
            const bool heavier = !usual && (heaviest > reference + 4.f || (reference == -INFINITY && heaviest > reference));
            if (__any_sync(kAllLanes, up || heavier)) {
              const float to = up ? best : top;
              const float down = up ? exp2f(top - to) : 1.f;
              total *= down;
              top = to;
              float by = down;
              if (!usual) {
                by = heavier ? exp2f(reference - heaviest) : 1.f;
                if (heavier) reference = heaviest;
              }
              if (step > 0) {
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
            // ---- the weights
            const float base = top == -INFINITY ? 0.f : top;
            float sum0 = 0.f, sum1 = 0.f;
            if (usual && !masked && a.runs) {
              const float unit = __uint_as_float(static_cast<uint32_t>(127 + 6 - exponent) << 23);
#pragma unroll 2
              for (int c = 0; c < 8; ++c) {
                const float by = note.k[c * 16] * unscale, vs = note.v[c * 16] * unit;
                float x[16];
                tmem_ld16(s_at + c * 16, x);
                tmem_wait_ld(x);
                uint32_t w[8];
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
                tmem_st8(s_at + c * 8, w);
              }
            } else {
              const float unit = __uint_as_float(static_cast<uint32_t>(127 + 6 - exponent) << 23);
              const float heavy = reference == -INFINITY ? 0.f : reference;
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {
                float x[16];
                tmem_ld16(s_at + c * 16, x);
                tmem_wait_ld(x);
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float vs = note.v[c * 16 + i];
                  float p = 0.f, y = 0.f;
                  if (!(vs < 0.f) && c * 16 + i < seen) {
                    const float t = x[i] * note.k[c * 16 + i] * unscale;
                    p = exp2_approx(t - base);
                    y = usual ? p * vs * unit : exp2_approx(t + log2f(vs) - heavy + 6.f);
                  }
                  sum0 += p;
                  x[i] = y;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = pack_f16x2(x[2 * i], x[2 * i + 1]);
                tmem_st8(s_at + c * 8, w);
              }
            }
            total += sum0 + sum1;
            tmem_wait_st();
          }
          tc_fence_before();
          arrive(&m.weights[slot]);
        }
        if (!going || !wait(&m.done[slot], done_turn & 1)) {
          going = false;
          break;
        }
        ++done_turn;
        tc_fence_after();
        // ---- the fragment's outputs
        if (warp_used) {
          const int64_t pairs = static_cast<int64_t>(a.rows) * a.heads, own_place = static_cast<int64_t>(token) * a.heads + head;
          int64_t place;
          if (f.first > 0) {
            place = a.at.starts + blockIdx.x * static_cast<int64_t>(kBlockRows) + slot * kSlotRows + row_in_slot;
          } else if (f.split && slot == 1) {
            place = a.at.copies + static_cast<int64_t>(it.extra) * a.cache.kv_heads + static_cast<int64_t>(f.kv) * it.rows + r;
          } else {
            place = it.prefix != 0 ? own_place : pairs + own_place;
          }
          // 2^(reference - top - 6) / total, in the usual case 2^(E - 6) / total.
          const float lift = usual ? static_cast<float>(exponent) : reference - top;
          const float by = total > 0.f || total != total ? exp2f(lift - 6.f) / total : 0.f;
          float4* out = reinterpret_cast<float4*>(a.part_out() + place * DIM);
#pragma unroll 1
          for (int c = 0; c < DIM; c += 16) {
            float o[16];
            tmem_ld16(o_at + c, o);
            tmem_wait_ld(o);
            if (used) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                out[c / 4 + i] = make_float4(o[4 * i] * by, o[4 * i + 1] * by, o[4 * i + 2] * by, o[4 * i + 3] * by);
              }
            }
          }
          if (used) a.part_lse()[place] = total == 0.f ? -INFINITY : top + log2f(total);
        }
        tc_fence_before();
      } else if (used) {
        // A fragment of one tile, all of it the other slot's.
        const int64_t place = f.first > 0 ? a.at.starts + blockIdx.x * static_cast<int64_t>(kBlockRows) + slot * kSlotRows + row_in_slot
                                          : a.at.copies + static_cast<int64_t>(it.extra) * a.cache.kv_heads +
                                                static_cast<int64_t>(f.kv) * it.rows + r;
        a.part_lse()[place] = -INFINITY;
      }
      tiles_before += f.last - f.first;
    }
  } else if (warp < kMmaWarp) {
    // ==================================================== keys and values
    // A warp widens 16 of a tile's rows, 16 codes a lane at a time; lanes 0 to 15
    // know the places of its rows. Codes are on their way a tile ahead.
    constexpr int kLanes = DIM / 16;        // to a row
    constexpr int kAtOnce = 32 / kLanes;    // rows
    constexpr int kTurns = 16 / kAtOnce;
    const int w = warp - 8;
    const int known_row = kAtOnce * w + (lane & (kAtOnce - 1)) + kAtOnce * kLoadWarps * ((lane & 15) / kAtOnce);
    struct Batch {
      uint4 k[kTurns], v[kTurns];
      float by, vs;
      bool any;
    };
    Batch batch[2];
    int32_t tile = 0, entry = 0;
    bool more = walk.next(a, f), bad = false;
    if (more) tile = f.first;
    auto page_of = [&](int32_t key) { return fastdiv(static_cast<uint32_t>(key), a.cache.block); };
    auto fetch = [&]() {  // the table's entry for this lane's row of the next tile
      const uint32_t page = min(page_of(f.item.key_begin + tile * kSharedTile + known_row), a.table_width - 1);
      entry = load_int(a.table + f.item.table_row * static_cast<int64_t>(a.table_width) + page);
    };
    auto issue = [&](Batch& b) {
      b.any = more;
      if (!more) return;
      const int32_t key = f.item.key_begin + tile * kSharedTile + known_row;
      const uint32_t page = page_of(key), offset = key - page * a.cache.block.divisor, block = entry;
      const bool wanted = key >= f.item.key_first && key < f.item.key_end;
      const bool good = wanted && page < a.table_width && block < a.cache.num_blocks;
      bad = bad || (wanted && !good);
      const int64_t k_place = good ? block * a.cache.k_block + offset * a.cache.k_token + f.kv * a.cache.k_head : -1;
      const int64_t v_place = block * a.cache.v_block + offset * a.cache.v_token + f.kv * a.cache.v_head;
      b.by = 0.f;
      b.vs = -1.f;
      if (good) {
        const int64_t s = static_cast<int64_t>(block) * a.cache.kv_heads + f.kv;
        b.by = __ldcg(a.cache.k_scale + s) * a.scale_log2;
        b.vs = __ldcg(a.cache.v_scale + s);
      }
      const int piece = lane & (kLanes - 1);
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int from = lane / kLanes + kAtOnce * i;
        const int64_t kp = __shfl_sync(kAllLanes, k_place, from), vp = __shfl_sync(kAllLanes, v_place, from);
        b.k[i] = b.v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (kp >= 0) {
          b.k[i] = __ldcg(reinterpret_cast<const uint4*>(a.cache.k + kp) + piece);
          b.v[i] = __ldcg(reinterpret_cast<const uint4*>(a.cache.v + vp) + piece);
        }
      }
      if (++tile == f.last) {
        more = walk.next(a, f);
        if (more) tile = f.first;
      }
      if (more) fetch();
    };
    uint32_t turn = 0;
    auto widen_to = [&](uint32_t to, const uint4 (&codes)[kTurns]) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const uint32_t row = kAtOnce * w + lane / kLanes + kAtOnce * kLoadWarps * i, piece = 2 * (lane & (kLanes - 1));
        const uint32_t c[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[2 * k] = e4m3x2_to_f16x2(static_cast<uint16_t>(c[k] & 0xffffu));
          h[2 * k + 1] = e4m3x2_to_f16x2(static_cast<uint16_t>(c[k] >> 16));
        }
        // The second half of a row goes the other way round, so that eight
        // lanes reach all banks.
        if (piece >= 8) {
          st_shared_v4(to + tile_place(row, piece + 1), h[4], h[5], h[6], h[7]);
          st_shared_v4(to + tile_place(row, piece), h[0], h[1], h[2], h[3]);
        } else {
          st_shared_v4(to + tile_place(row, piece), h[0], h[1], h[2], h[3]);
          st_shared_v4(to + tile_place(row, piece + 1), h[4], h[5], h[6], h[7]);
        }
      }
    };
    auto step = [&](Batch& now, Batch& next) {
      issue(next);
      if (!now.any) return false;
      const uint32_t stage = turn % kStages, parity = (turn / kStages & 1) ^ 1;
      if (!wait(&m.k_free[stage], parity)) return false;
      widen_to(smem_addr(m.k[stage]), now.k);
      Note& note = m.note[turn % kNotes];
      const int32_t e = static_cast<int32_t>(__float_as_uint(now.vs) >> 23 & 0xff);
      const bool counts = now.vs > 0.f && e != 255;  // neither 0, nor NaN, nor a key that does not count
      const int32_t most = __reduce_max_sync(kAllLanes, counts ? e - 127 : -1000);
      const int32_t least = __reduce_min_sync(kAllLanes, counts ? e - 127 : 1000);
      const bool holes = __any_sync(kAllLanes, now.vs < 0.f);
      if (lane < 16) {
        note.k[known_row] = now.by;
        note.v[known_row] = now.vs;
      }
      if (lane == 0) note.seen[w] = make_int4(most, least, holes ? 1 : 0, 0);
      fence_proxy_async();
      arrive(&m.k_full[stage]);
      if (!wait(&m.v_free[stage], parity)) return false;
      widen_to(smem_addr(m.v[stage]), now.v);
      fence_proxy_async();
      arrive(&m.v_full[stage]);
      ++turn;
      return true;
    };
    if (more) {
      fetch();
      issue(batch[0]);
      while (step(batch[0], batch[1]) && step(batch[1], batch[0])) {
      }
    }
    if (bad) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
  } else {
    // ==================================================== MMAs
    constexpr uint32_t kScoreDesc = mma_descriptor(128, kSharedTile, 0, false, false);
    constexpr uint32_t kOutDesc = mma_descriptor(128, DIM, 0, false, true);
    constexpr uint32_t kChunk = kSharedTile * 128;  // bytes of 64 columns of a tile
    const bool leader = elect_one();
    uint32_t k_turn = 0, v_turn = 0, weights_turn[2] = {0, 0}, queries_turn[2] = {0, 0};
    bool going = true;
    while (going && walk.next(a, f)) {
      const int32_t ops = f.split ? f.last - f.first : 2 * (f.last - f.first);
      for (int32_t n = 0; n <= ops; ++n) {
        if (n < ops) {  // scores
          const int slot = n & 1;
          const uint32_t stage = k_turn % kStages;
          if ((f.split || slot == 0) && !wait(&m.k_full[stage], k_turn / kStages & 1)) going = false;
          if (going && n < 2) going = wait(&m.queries[slot], queries_turn[slot]++ & 1);
          if (!going) break;
          tc_fence_after();
          if (leader) {
            const uint64_t qd = smem_descriptor(smem_addr(m.q[slot]), 16, 1024, kSwizzle128);
            const uint64_t kd = smem_descriptor(smem_addr(m.k[stage]), 16, 1024, kSwizzle128);
#pragma unroll
            for (int k = 0; k < DIM / 16; ++k) {
              const uint32_t at = (k / 4 * kChunk + k % 4 * 32) >> 4;
              mma_f16(tmem + kScoresAt + slot * kSharedTile, qd + at, kd + at, kScoreDesc, k > 0);
            }
            if (f.split || slot == 1) mma_commit(smem_addr(&m.k_free[stage]));
            mma_commit(smem_addr(&m.scores[slot]));
          }
          __syncwarp();
          if (f.split || slot == 1) ++k_turn;
        }
        if (n > 0) {  // outputs of the one before
          const int slot = (n - 1) & 1;
          const uint32_t stage = v_turn % kStages;
          if (!wait(&m.weights[slot], weights_turn[slot]++ & 1)) going = false;
          if (going && (f.split || slot == 0)) going = wait(&m.v_full[stage], v_turn / kStages & 1);
          if (!going) break;
          tc_fence_after();
          if (leader) {
            const uint64_t vd = smem_descriptor(smem_addr(m.v[stage]), kChunk, 1024, kSwizzle128);
#pragma unroll
            for (int k = 0; k < kSharedTile / 16; ++k) {
              mma_f16_tmem(tmem + slot * DIM, tmem + kScoresAt + slot * kSharedTile + k * 8, vd + (k * 2048 >> 4), kOutDesc,
                           k > 0 || n > 2);
            }
            if (f.split || slot == 1) mma_commit(smem_addr(&m.v_free[stage]));
            if (n + 1 >= ops) mma_commit(smem_addr(&m.done[slot]));
          }
          __syncwarp();
          if (f.split || slot == 1) ++v_turn;
        }
      }
    }
    if (!going) {  // gave up: let what was issued finish before the memory goes
      if (leader) {
        mma_commit(smem_addr(&m.drained));
        const long long begin = clock64();
        while (!mbar_try(smem_addr(&m.drained), 0) && clock64() - begin < 4000000000LL) {
        }
      }
      __syncwarp();
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
  constexpr int bytes = static_cast<int>(sizeof(Memory<DIM>)) + 1024;
  static_assert(bytes <= 227 * 1024, "shared memory");
  void (*fn)(SharedArgs) = shared_kernel<T, DIM>;
  const int rc = allow_launch(reinterpret_cast<const void*>(fn), bytes, granted);
  if (rc != SILKERN_OK) return rc;
  return launch_pdl(fn, grid, kThreads, bytes, 1, stream, a);
}

}  // namespace shared
}  // namespace silkern
