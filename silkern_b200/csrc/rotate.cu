// Queries and new keys before they are asked and stored: a norm of each head's
// first columns, and the rotation of some of its columns by position.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "cache_checks.cuh"
#include "host.cuh"
#include "ptx.cuh"
#include "silkern_b200.h"

namespace silkern {

namespace {

constexpr int kRotateThreads = 256;
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
  int32_t group, slots;               // lanes to a head; pieces of 8 columns that pair up
  int32_t heads_a_cta;
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

// The place in a head's columns of a thread's two pieces of 8. The first
// pairs / 8 slots of a head rotate in halves: the piece and the one that it is
// paired with. Other slots hold pieces half the slots apart, in the order that
// leaves those out; -1: none.
struct Pieces {
  int32_t a, b;
  bool rotates;  // a with b
};
__device__ __forceinline__ Pieces pieces_of(const RotateArgs& g, int32_t slot) {
  const int32_t total = g.dim >> 3;
  if (g.interleaved) {
    const int32_t b = slot + g.slots;
    return {slot * 8, b < total ? b * 8 : -1, false};
  }
  const int32_t turned = g.pairs >> 3, first = g.start >> 3;
  if (slot < turned) return {(first + slot) * 8, (first + turned + slot) * 8, true};
  const int32_t rest = total - 2 * turned, plain = slot - turned, half = (rest + 1) >> 1;
  auto place = [&](int32_t p) { return (p < first ? p : p + 2 * turned) * 8; };
  return {place(plain), plain + half < rest ? place(plain + half) : -1, false};
}

// One CTA for a token and up to heads_a_cta of its heads, `group` lanes to a
// head, N slots of two pieces of 8 columns to a lane. The token's cos and sin
// are worked out once, for all of the CTA's heads, and the weights widened,
// while the first heads are on their way. Every element is read and written
// once.
template <typename T, int N>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(const __grid_constant__ RotateArgs g) {
  __shared__ __align__(16) float table[2][kMostColumns / 2];  // cos, sin
  __shared__ __align__(16) float weights[2][kMostColumns];
  pdl_wait();
  pdl_launch_dependents();
  const int32_t token = blockIdx.x;
  const int32_t lane = threadIdx.x % g.group, team = threadIdx.x / g.group, teams = kRotateThreads / g.group;
  const int32_t first = blockIdx.y * g.heads_a_cta, last = min(first + g.heads_a_cta, g.all_heads);
  auto set_of = [&](int32_t head) -> const HeadSet& { return g.set[head < g.set[0].heads ? 0 : 1]; };
  uint4 raw[N][2];
  auto fetch = [&](int32_t head) {
    const HeadSet& s = set_of(head);
    const int32_t h = head < g.set[0].heads ? head : head - g.set[0].heads;
    const T* p = static_cast<const T*>(s.in) + token * s.in_token + h * s.in_head;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int32_t slot = lane + n * g.group;
      raw[n][0] = raw[n][1] = make_uint4(0u, 0u, 0u, 0u);
      if (slot < g.slots) {
        const Pieces at = pieces_of(g, slot);
        raw[n][0] = load_wide(p + at.a);
        if (at.b >= 0) raw[n][1] = load_wide(p + at.b);
      }
    }
  };
  int32_t head = first + team;
  if (head < last) fetch(head);
  const int32_t position = g.positions[token];
  for (int32_t i = threadIdx.x; i < g.pairs; i += kRotateThreads) {
    const float2 t = turn(position, g.frequencies[i], g.amplitude);
    table[0][i] = t.x;
    table[1][i] = t.y;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 0 ? first >= g.set[0].heads : last <= g.set[0].heads) continue;
    for (int32_t i = threadIdx.x; i < g.set[k].norm; i += kRotateThreads) {
      weights[k][i] = g.weights_f32 ? static_cast<const float*>(g.set[k].weight)[i]
                                    : static_cast<float>(static_cast<const T*>(g.set[k].weight)[i]);
    }
  }
  __syncthreads();
  // Lanes of a head share a warp; a warp's heads run out together or not, so
  // that every lane takes part in the exchanges.
  for (int32_t base = first; base < last; base += teams, head += teams) {
    const bool live = head < last;
    const HeadSet& s = set_of(live ? head : first);
    const int k = &s == &g.set[0] ? 0 : 1;
    if (base > first && live) fetch(head);
    float x[N][2][8];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      unpack8<T>(raw[n][0], x[n][0]);
      unpack8<T>(raw[n][1], x[n][1]);
    }
    if (g.set[0].norm | g.set[1].norm) {
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int32_t slot = lane + n * g.group;
        if (slot >= g.slots) continue;
        const Pieces at = pieces_of(g, slot);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (at.a + i < s.norm) sum = fmaf(x[n][0][i], x[n][0][i], sum);
          if (at.b >= 0 && at.b + i < s.norm) sum = fmaf(x[n][1][i], x[n][1][i], sum);
        }
      }
      for (int d = g.group >> 1; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
      const float r = s.norm > 0 ? rsqrtf(sum / static_cast<float>(s.norm) + g.eps) : 1.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int32_t slot = lane + n * g.group;
        if (slot >= g.slots) continue;
        const Pieces at = pieces_of(g, slot);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (at.a + i < s.norm) x[n][0][i] *= r * weights[k][at.a + i];
          if (at.b >= 0 && at.b + i < s.norm) x[n][1][i] *= r * weights[k][at.b + i];
        }
      }
    }
    if (!live) continue;
    const int32_t h = head < g.set[0].heads ? head : head - g.set[0].heads;
    T* out = static_cast<T*>(s.out) + token * s.out_token + h * s.out_head;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int32_t slot = lane + n * g.group;
      if (slot >= g.slots) continue;
      const Pieces at = pieces_of(g, slot);
      if (at.rotates) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = table[0][slot * 8 + i], z = table[1][slot * 8 + i];
          const float a = x[n][0][i], b = x[n][1][i];
          x[n][0][i] = a * c - b * z;
          x[n][1][i] = b * c + a * z;
        }
      } else if (g.interleaved) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int32_t at_pair = ((e == 0 ? at.a : at.b) - g.start) >> 1;
          if ((e == 1 && at.b < 0) || at_pair < 0 || at_pair >= g.pairs) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float c = table[0][at_pair + i], z = table[1][at_pair + i];
            const float a = x[n][e][2 * i], b = x[n][e][2 * i + 1];
            x[n][e][2 * i] = a * c - b * z;
            x[n][e][2 * i + 1] = b * c + a * z;
          }
        }
      }
      *reinterpret_cast<uint4*>(out + at.a) = pack8<T>(x[n][0]);
      if (at.b >= 0) *reinterpret_cast<uint4*>(out + at.b) = pack8<T>(x[n][1]);
    }
  }
}

// The same by single elements, a warp to a head, for columns, strides or
// addresses that no pieces of 16 bytes fit.
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
  switch (each) {
    case 1: return rotate_kernel<T, 1>;
    case 2: return rotate_kernel<T, 2>;
    case 3: return rotate_kernel<T, 3>;
    case 4: return rotate_kernel<T, 4>;
    default: return rotate_kernel<T, 5>;
  }
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
    g.all_heads += s.heads;
    wide = wide && (s.in_token | s.in_head | s.out_token | s.out_head) % 8 == 0 &&
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
  int each = 0, teams = kRotateThreads / 32;
  if (wide) {
    const int total = dim / 8, turned = g.interleaved ? 0 : pairs / 8;
    g.slots = turned + (total - 2 * turned + 1) / 2;
    // Lanes to a head: of the powers of two with at most five slots to a lane,
    // the one with the fewest slots left empty, and the most lanes among equals.
    int least = 0;
    for (int group = 32; group >= 1; group >>= 1) {
      const int n = (g.slots + group - 1) / group;
      if (n <= 5 && (each == 0 || n * group < least)) {
        each = n;
        g.group = group;
        least = n * group;
      }
    }
    teams = kRotateThreads / g.group;
  }
  // A token's heads in one CTA, unless few tokens leave SMs without work.
  int64_t parts = 1;
  while (parts * teams < g.all_heads && parts * tokens < 2 * 148) ++parts;
  g.heads_a_cta = static_cast<int32_t>((g.all_heads + parts - 1) / parts);
  parts = (g.all_heads + g.heads_a_cta - 1) / g.heads_a_cta;
  void (*fn)(RotateArgs) = type == SILKERN_BF16
                               ? (wide ? rotate_for<__nv_bfloat16>(each) : rotate_narrow_kernel<__nv_bfloat16>)
                               : (wide ? rotate_for<__half>(each) : rotate_narrow_kernel<__half>);
  return launch_pdl_grid(fn, dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(parts), 1), kRotateThreads, 0, 1,
                         static_cast<cudaStream_t>(stream), g);
}
