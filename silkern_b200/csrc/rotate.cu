// Queries and new keys before they are asked and stored: a norm of each head's
// first columns, and the rotation of some of its columns by position.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache_checks.cuh"
#include "host.cuh"
#include "ptx.cuh"
#include "silkern_b200.h"

namespace silkern {

namespace {

constexpr int kRotateThreads = 256;  // at most
constexpr int kMostColumns = SILKERN_MOST_COLUMNS;

struct HeadSet {
  const void* in;
  void* out;
  const void* weight;
  int64_t in_token, in_head, out_token, out_head;  // elements
  int32_t heads, norm;
};

struct RotateArgs {
  HeadSet set[2];
  const int32_t* positions;
  const float* frequencies;
  int32_t tokens, dim, pairs, start;  // pairs: of rotary columns, the first in column `start`
  int32_t all_heads;                  // of both sets
  int32_t normed[2];                  // the heads [normed[0], normed[1]) of them have a norm
  int32_t group;                      // lanes to a normed head
  FastDiv slots;                      // by a head's slots of two pieces of 8 columns
  int32_t heads_a_cta, tokens_a_cta;  // all heads where there are several tokens
  FastDiv by_normed, by_plain;        // then: by a token's normed heads, by its other heads' slots
  bool interleaved, weights_f32;
  float amplitude, eps;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = __uint_as_float(r[i] << 16);
      x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __half2 p = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ uint4 load_wide(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// cos and sin of position * frequency, times the amplitude. In turns and in
// double: a float's 24 bits hold an angle of 10^5 to 0.004, these to 2^-36 of a
// turn at least where positions are below 2^17. What is left of the turn after
// the whole ones fits a float.
__device__ __forceinline__ float2 turn(int32_t position, float frequency, float amplitude) {
  const double turns = static_cast<double>(position) * (static_cast<double>(frequency) * 0.15915494309189533577);
  float s, c;
  sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c * amplitude, s * amplitude);
}

// The place in a head's columns of a slot's two pieces of 8. The first pairs / 8
// slots of a head rotate in halves: the piece and the one that it is paired with.
// Other slots hold pieces half the slots apart, in the order that leaves those
// out; -1: none.
struct Pieces {
  int32_t a, b;
  bool rotates;  // a with b
};
__device__ __forceinline__ Pieces pieces_of(const RotateArgs& g, int32_t slot) {
  const int32_t total = g.dim >> 3;
  if (g.interleaved) {
    const int32_t b = slot + static_cast<int32_t>(g.slots.divisor);
    return {slot * 8, b < total ? b * 8 : -1, false};
  }
  const int32_t turned = g.pairs >> 3, first = g.start >> 3;
  if (slot < turned) return {(first + slot) * 8, (first + turned + slot) * 8, true};
  const int32_t rest = total - 2 * turned, plain = slot - turned, half = (rest + 1) >> 1;
  auto place = [&](int32_t p) { return (p < first ? p : p + 2 * turned) * 8; };
  return {place(plain), plain + half < rest ? place(plain + half) : -1, false};
}

struct Tables {
  float cos[kMostColumns / 2], sin[kMostColumns / 2];
  float weight[2][kMostColumns];
};
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void rotate_slot(const RotateArgs& g, const Tables& t, int32_t row, int32_t slot, const Pieces& at, float (&a)[8],
                                            float (&b)[8]) {
  if (at.rotates) {
    float c[8], s[8];
    load8(t.cos + row + slot * 8, c);
    load8(t.sin + row + slot * 8, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  } else if (g.interleaved) {
    auto turn = [&](int32_t column, float (&x)[8]) {
      const int32_t pair = (column - g.start) >> 1;
      if (column < g.start || pair >= g.pairs) return;
      const float4 c = *reinterpret_cast<const float4*>(t.cos + row + pair), s = *reinterpret_cast<const float4*>(t.sin + row + pair);
      const float cs[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x0 = x[2 * i], x1 = x[2 * i + 1];
        x[2 * i] = x0 * cs[i] - x1 * ss[i];
        x[2 * i + 1] = x1 * cs[i] + x0 * ss[i];
      }
    };
    turn(at.a, a);
    if (at.b >= 0) turn(at.b, b);
  }
}

// One CTA for a token and up to heads_a_cta of its heads, or for all heads of a few
// tokens. The tokens' cos and sin are worked out once, for all of the CTA's heads,
// and the weights widened. Heads with a norm take `group` lanes each and N slots a
// lane; the slots of the others are dealt out one by one, two a thread on their way
// at once. Every element is read and written once, 16 bytes at a time. Bound by
// memory and, with norms, by instruction issue: 8192 tokens of 72 normed heads of
// 128 columns (302 MB) 60 us, 5.0 TB/s; 1001 tokens of 129 heads of 576, 64 of them
// rotary (298 MB), 57 us, 5.2 TB/s. Four CTAs to an SM (64 registers): with
// three (80) or five (48, spilled) 64 us each.
template <typename T, int N>
__global__ void __launch_bounds__(kRotateThreads, 4) rotate_kernel(const __grid_constant__ RotateArgs g) {
  __shared__ __align__(16) Tables tables;
  pdl_wait();
  pdl_launch_dependents();
  const int32_t token0 = blockIdx.x * g.tokens_a_cta, threads = blockDim.x;
  const int32_t tokens = min(g.tokens_a_cta, g.tokens - token0);
  const int32_t first = blockIdx.y * g.heads_a_cta, last = min(first + g.heads_a_cta, g.all_heads);
  const int32_t q_heads = g.set[0].heads;
  auto source = [&](int32_t token, int32_t head) {
    const HeadSet& s = g.set[head < q_heads ? 0 : 1];
    return static_cast<const T*>(s.in) + (token0 + token) * s.in_token + (head < q_heads ? head : head - q_heads) * s.in_head;
  };
  auto target = [&](int32_t token, int32_t head) {
    const HeadSet& s = g.set[head < q_heads ? 0 : 1];
    return static_cast<T*>(s.out) + (token0 + token) * s.out_token + (head < q_heads ? head : head - q_heads) * s.out_head;
  };
  const int32_t normed_first = max(first, g.normed[0]), normed_last = min(last, g.normed[1]);
  const int32_t lane = threadIdx.x % g.group, team = threadIdx.x / g.group, teams = threads / g.group;
  Pieces at[N];
  uint4 raw[N][2];
  // Units: a token and one of its normed heads.
  const int32_t normed = max(normed_last - normed_first, 0), units = tokens * normed;
  auto token_of = [&](int32_t unit) { return tokens > 1 ? static_cast<int32_t>(fastdiv(unit, g.by_normed)) : 0; };
  auto fetch = [&](int32_t unit) {
    const int32_t token = token_of(unit);
    const T* p = source(token, normed_first + unit - token * normed);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      raw[n][0] = raw[n][1] = make_uint4(0u, 0u, 0u, 0u);
      if (at[n].a >= 0) raw[n][0] = load_wide(p + at[n].a);
      if (at[n].b >= 0) raw[n][1] = load_wide(p + at[n].b);
    }
  };
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int32_t slot = lane + n * g.group;
    at[n] = slot < static_cast<int32_t>(g.slots.divisor) ? pieces_of(g, slot) : Pieces{-1, -1, false};
  }
  int32_t unit = team;
  if (unit < units) fetch(unit);
  // Heads without a norm: those below normed_first and from normed_last on.
  const int32_t below = min(last, g.normed[0]) - first, slots = g.slots.divisor;
  const int32_t before = max(below, 0), behind_first = max(first, g.normed[1]), plain = before + max(last - behind_first, 0);
  const int32_t each = plain * slots, all = tokens * each;
  constexpr int kAtOnce = 2;
  struct Dealt {
    int32_t token, head, slot;  // slot -1: none
  };
  uint4 ahead[kAtOnce][2];
  Dealt dealt[kAtOnce];
  auto deal = [&](int32_t i0) {
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const int32_t i = i0 + n * threads;
      ahead[n][0] = ahead[n][1] = make_uint4(0u, 0u, 0u, 0u);
      dealt[n] = Dealt{0, 0, -1};
      if (i < all) {
        const int32_t token = tokens > 1 ? static_cast<int32_t>(fastdiv(i, g.by_plain)) : 0;
        const int32_t j = i - token * each, h = static_cast<int32_t>(fastdiv(j, g.slots));
        dealt[n] = Dealt{token, h < before ? first + h : behind_first + h - before, j - h * slots};
        const Pieces piece = pieces_of(g, dealt[n].slot);
        const T* p = source(token, dealt[n].head);
        ahead[n][0] = load_wide(p + piece.a);
        if (piece.b >= 0) ahead[n][1] = load_wide(p + piece.b);
      }
    }
  };
  if (units == 0) deal(threadIdx.x);
  for (int32_t i = threadIdx.x; i < g.pairs * tokens; i += threads) {
    const int32_t token = i / g.pairs;
    const float2 t = turn(g.positions[token0 + token], g.frequencies[i - token * g.pairs], g.amplitude);
    tables.cos[i] = t.x;
    tables.sin[i] = t.y;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 0 ? first >= q_heads : last <= q_heads) continue;
    for (int32_t i = threadIdx.x; i < g.set[k].norm; i += threads) {
      tables.weight[k][i] = g.weights_f32 ? static_cast<const float*>(g.set[k].weight)[i]
                                          : static_cast<float>(static_cast<const T*>(g.set[k].weight)[i]);
    }
  }
  __syncthreads();
  // Lanes of a head share a warp; all of a warp goes as often round, so that every
  // lane takes part in the exchanges.
  for (int32_t base = 0; base < units; base += teams, unit += teams) {
    const bool live = unit < units;
    const int32_t token = live ? token_of(unit) : 0, head = normed_first + unit - token * normed;
    const int k = live && head >= q_heads ? 1 : 0;
    const int32_t norm = g.set[k].norm;
    float x[N][2][8], sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        unpack8<T>(raw[n][e], x[n][e]);
        const int32_t column = e == 0 ? at[n].a : at[n].b;
        if (column >= 0 && column < norm) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(x[n][e][i], x[n][e][i], sum);
        }
      }
    }
    if (unit + teams < units) fetch(unit + teams);
    for (int d = g.group >> 1; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
    if (!live) continue;
    const float r = rsqrtf(sum / static_cast<float>(norm) + g.eps);
    T* out = target(token, head);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (at[n].a < 0) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int32_t column = e == 0 ? at[n].a : at[n].b;
        if (column >= 0 && column < norm) {
          float w[8];
          load8(tables.weight[k] + column, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[n][e][i] *= r * w[i];
        }
      }
      rotate_slot(g, tables, token * g.pairs, lane + n * g.group, at[n], x[n][0], x[n][1]);
      *reinterpret_cast<uint4*>(out + at[n].a) = pack8<T>(x[n][0]);
      if (at[n].b >= 0) *reinterpret_cast<uint4*>(out + at[n].b) = pack8<T>(x[n][1]);
    }
  }
  if (units > 0) deal(threadIdx.x);
  for (int32_t i0 = threadIdx.x; i0 < all; i0 += kAtOnce * threads) {
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const Dealt& d = dealt[n];
      if (d.slot < 0) continue;
      const Pieces piece = pieces_of(g, d.slot);
      float a[8], b[8];
      unpack8<T>(ahead[n][0], a);
      unpack8<T>(ahead[n][1], b);
      rotate_slot(g, tables, d.token * g.pairs, d.slot, piece, a, b);
      T* out = target(d.token, d.head);
      *reinterpret_cast<uint4*>(out + piece.a) = pack8<T>(a);
      if (piece.b >= 0) *reinterpret_cast<uint4*>(out + piece.b) = pack8<T>(b);
    }
    deal(i0 + kAtOnce * threads);
  }
}

// The same by single elements, a warp to a head, for columns, strides or
// addresses that no pieces of 16 bytes fit. Bound by the loads and stores of 2 bytes:
// 8192 tokens of 72 normed heads of 128 columns, one element off alignment, 199 us
// (68 in pieces, timed alike: with cold caches), 1001 tokens of 129 latent heads 186 (64).
template <typename T>
__global__ void __launch_bounds__(kRotateThreads) rotate_narrow_kernel(const __grid_constant__ RotateArgs g) {
  __shared__ float table[2][kMostColumns / 2];
  pdl_wait();
  pdl_launch_dependents();
  const int32_t token = blockIdx.x, lane = threadIdx.x & 31;
  const int32_t position = g.positions[token];
  for (int32_t i = threadIdx.x; i < g.pairs; i += kRotateThreads) {
    const float2 t = turn(position, g.frequencies[i], g.amplitude);
    table[0][i] = t.x;
    table[1][i] = t.y;
  }
  __syncthreads();
  const int32_t first = blockIdx.y * g.heads_a_cta, last = min(first + g.heads_a_cta, g.all_heads);
  for (int32_t head = first + (threadIdx.x >> 5); head < last; head += kRotateThreads / 32) {
    const HeadSet& s = g.set[head < g.set[0].heads ? 0 : 1];
    const int32_t h = head < g.set[0].heads ? head : head - g.set[0].heads;
    const T* in = static_cast<const T*>(s.in) + token * s.in_token + h * s.in_head;
    T* out = static_cast<T*>(s.out) + token * s.out_token + h * s.out_head;
    float r = 1.f;
    if (s.norm > 0) {
      float sum = 0.f;
      for (int32_t i = lane; i < s.norm; i += 32) {
        const float x = static_cast<float>(in[i]);
        sum = fmaf(x, x, sum);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
      r = rsqrtf(sum / static_cast<float>(s.norm) + g.eps);
    }
    auto normed = [&](int32_t i) {
      const float x = static_cast<float>(in[i]);
      if (i >= s.norm) return x;
      return x * (r * (g.weights_f32 ? static_cast<const float*>(s.weight)[i]
                                     : static_cast<float>(static_cast<const T*>(s.weight)[i])));
    };
    // A lane reads both elements of a pair before it writes them, so that out
    // may be in.
    for (int32_t i = lane; i < g.pairs; i += 32) {
      const int32_t at = g.start + (g.interleaved ? 2 * i : i), to = g.interleaved ? at + 1 : at + g.pairs;
      const float a = normed(at), b = normed(to), c = table[0][i], z = table[1][i];
      out[at] = static_cast<T>(a * c - b * z);
      out[to] = static_cast<T>(b * c + a * z);
    }
    for (int32_t i = lane; i < g.dim - 2 * g.pairs; i += 32) {
      const int32_t at = i < g.start ? i : i + 2 * g.pairs;
      out[at] = static_cast<T>(normed(at));
    }
  }
}

template <typename T>
void (*rotate_for(int each))(RotateArgs) {
  return each == 1 ? rotate_kernel<T, 1> : rotate_kernel<T, 2>;
}

Place place_of_heads(const void* base, int32_t dim, int64_t tokens, int64_t token, int32_t heads, int64_t head) {
  return Place(base, 2 * static_cast<int64_t>(dim)).along(tokens, 2 * token).along(heads, 2 * head);
}

}  // namespace
}  // namespace silkern

using namespace silkern;

extern "C" int silkern_rotate_heads_v1(const silkern_heads_v1* q, const silkern_heads_v1* k, int32_t type, int64_t tokens,
                                       int32_t dim, const int32_t* positions, const float* frequencies, int32_t pairs,
                                       int32_t rotary_start, int32_t interleaved, int32_t weights_f32, float amplitude,
                                       float eps, void* stream) {
  if (!q || !q->in || !q->out || !positions || !frequencies) return SILKERN_E_NULL;
  if (k != nullptr && (!k->in || !k->out)) return SILKERN_E_NULL;
  if (type != SILKERN_BF16 && type != SILKERN_F16) return SILKERN_E_TYPE;
  if (tokens < 1 || tokens > 0x7fffffff || dim < 1 || dim > kMostColumns) return SILKERN_E_SHAPE;
  if (pairs < 1 || rotary_start < 0 || pairs > dim / 2 || rotary_start > dim - 2 * pairs) return SILKERN_E_ROTARY;
  if (!std::isfinite(amplitude) || !std::isfinite(eps) || eps < 0.f) return SILKERN_E_ROTARY;
  RotateArgs g{};
  const silkern_heads_v1* sets[2] = {q, k};
  bool wide = (dim | rotary_start) % 8 == 0 && pairs % (interleaved ? 4 : 8) == 0;
  for (int i = 0; i < 2 && sets[i] != nullptr; ++i) {
    const silkern_heads_v1& s = *sets[i];
    if (s.heads < 1 || s.heads > 65535) return SILKERN_E_HEADS;
    if (s.norm_columns < 0 || s.norm_columns > dim) return SILKERN_E_ROTARY;
    if (s.norm_columns > 0 && s.weight == nullptr) return SILKERN_E_NULL;
    g.set[i] = HeadSet{s.in, s.out, s.weight, s.in_token, s.in_head, s.out_token, s.out_head, s.heads, s.norm_columns};
    if (s.norm_columns > 0) {
      if (g.normed[1] == 0) g.normed[0] = g.all_heads;
      g.normed[1] = g.all_heads + s.heads;
    }
    g.all_heads += s.heads;
    wide = wide && s.norm_columns % 8 == 0 && (s.in_token | s.in_head | s.out_token | s.out_head) % 8 == 0 &&
           (reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out)) % 16 == 0;
  }
  // An output is its own input, element for element, or lies apart from every
  // buffer of the call.
  const Place small[2] = {Place(positions, 4 * tokens), Place(frequencies, 4 * static_cast<int64_t>(pairs))};
  for (int i = 0; i < 2 && sets[i] != nullptr; ++i) {
    const silkern_heads_v1& s = *sets[i];
    const Place out = place_of_heads(s.out, dim, tokens, s.out_token, s.heads, s.out_head);
    if (!single(out) || shares(out, small[0]) || shares(out, small[1])) return SILKERN_E_ALIAS;
    for (int j = 0; j < 2 && sets[j] != nullptr; ++j) {
      const silkern_heads_v1& o = *sets[j];
      const bool same = i == j && s.in == s.out && (tokens == 1 || s.in_token == s.out_token) &&
                        (s.heads == 1 || s.in_head == s.out_head);
      if (!same && shares(out, place_of_heads(o.in, dim, tokens, o.in_token, o.heads, o.in_head))) return SILKERN_E_ALIAS;
      if (i != j && shares(out, place_of_heads(o.out, dim, tokens, o.out_token, o.heads, o.out_head))) return SILKERN_E_ALIAS;
      if (o.norm_columns > 0 && shares(out, Place(o.weight, (weights_f32 ? 4 : 2) * static_cast<int64_t>(o.norm_columns)))) {
        return SILKERN_E_ALIAS;
      }
    }
  }
  g.positions = positions;
  g.frequencies = frequencies;
  g.tokens = static_cast<int32_t>(tokens);
  g.dim = dim;
  g.pairs = pairs;
  g.start = rotary_start;
  g.interleaved = interleaved != 0;
  g.weights_f32 = weights_f32 != 0;
  g.amplitude = amplitude;
  g.eps = eps;
  int each = 1, threads = kRotateThreads;
  int64_t in_turn = kRotateThreads / 32;  // heads of a CTA at once
  g.group = 32;
  if (wide) {
    const int total = dim / 8, turned = g.interleaved ? 0 : pairs / 8, slots = turned + (total - 2 * turned + 1) / 2;
    g.slots = make_fastdiv(static_cast<uint32_t>(slots));
    // Lanes to a normed head: of the powers of two with at most two slots to a lane
    // (three take registers that the others' occupancy needs: 76 us for 65 on 1001
    // tokens of 129 latent heads), the one with the fewest slots left empty, and the
    // most lanes among equals.
    int least = 0;
    for (int group = 32; group >= 1; group >>= 1) {
      const int n = (slots + group - 1) / group;
      if (n <= 2 && (least == 0 || n * group < least)) {
        each = n;
        g.group = group;
        least = n * group;
      }
    }
    in_turn = kRotateThreads / g.group;
  }
  // A token's heads in one CTA of at most 48 KB, unless few tokens leave SMs
  // without work.
  int64_t parts = (2 * int64_t{dim} * g.all_heads + 49151) / 49152;
  while (parts * in_turn < g.all_heads && parts * tokens < 2 * 148) ++parts;
  g.heads_a_cta = static_cast<int32_t>((g.all_heads + parts - 1) / parts);
  parts = (g.all_heads + g.heads_a_cta - 1) / g.heads_a_cta;
  const int32_t normed = g.normed[1] - g.normed[0];
  g.tokens_a_cta = 1;
  if (wide && parts == 1) {
    // Several tokens while a CTA has less than 48 KB of them, there is room for their
    // cos and sin, and six CTAs for each SM.
    const int64_t bytes = 2 * int64_t{dim} * g.all_heads;
    const int64_t most = std::min({(49152 + bytes - 1) / bytes, int64_t{kMostColumns / 2 / pairs}, tokens / (6 * 148)});
    g.tokens_a_cta = static_cast<int32_t>(std::max(most, int64_t{1}));
    g.by_normed = make_fastdiv(static_cast<uint32_t>(normed > 0 ? normed : 1));
    const int64_t plain = (g.all_heads - normed) * static_cast<int64_t>(g.slots.divisor);
    g.by_plain = make_fastdiv(static_cast<uint32_t>(plain > 0 ? plain : 1));
  }
  if (wide && normed > 0) {
    // As many threads as leave the fewest without a head in the last round (72
    // heads of 8 lanes: 192 threads, three rounds).
    const int64_t heads = int64_t{normed < g.heads_a_cta ? normed : g.heads_a_cta} * g.tokens_a_cta;
    int64_t best = 0;
    for (int candidate = kRotateThreads; candidate >= 128; candidate -= 32) {
      const int64_t teams = candidate / g.group, rounds = (heads + teams - 1) / teams;
      const int64_t filled = heads * 1000 / (rounds * teams);
      if (filled > best) {
        best = filled;
        threads = candidate;
      }
    }
  }
  void (*fn)(RotateArgs) = type == SILKERN_BF16
                               ? (wide ? rotate_for<__nv_bfloat16>(each) : rotate_narrow_kernel<__nv_bfloat16>)
                               : (wide ? rotate_for<__half>(each) : rotate_narrow_kernel<__half>);
  return launch_pdl_grid(fn, dim3(static_cast<unsigned>((tokens + g.tokens_a_cta - 1) / g.tokens_a_cta), static_cast<unsigned>(parts), 1), threads, 0, 1,
                         static_cast<cudaStream_t>(stream), g);
}
