// Attention over the 8-bit paged cache: selected slots, and a window with
// sinks through the block table.
//
//   out[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(softmax_scale * q[r, h] . k_j)
//   lse[r, h] = log sum_j p_j                 (natural log; -inf and out 0 where nothing is visible)
//
// One CTA for each (query row, head); the warps take the keys in turn and keep
// a running maximum, sum and output in float32 registers, joined at the end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "host.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "silkern_b200.h"

namespace silkern {
namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ float e4m3_to_float(uint8_t code) {
  __nv_fp8_e4m3 x;
  x.__x = code;
  return static_cast<float>(x);
}

template <typename T, int DK, int DV>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int KL = DK / 32, VL = DV / 32;
  __shared__ float shared_m[kWarps], shared_l[kWarps], shared_o[kWarps][DV];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.x % a.heads, item = blockIdx.x / a.heads, kv = head / a.heads_per_kv;
  KeyList keys;
  int row = item;
  if (a.slots != nullptr) {
    keys = selected_keys(a, item);
  } else {
    const QuerySpan s = find_span(a, item, a.one);
    if (s.count == 0) return;
    row = s.row;
    keys = window_keys(a, s);
  }
  const T* q = static_cast<const T*>(a.q) + row * a.q_row + head * a.q_head;
  float qr[KL], o[VL];
#pragma unroll
  for (int i = 0; i < KL; ++i) qr[i] = static_cast<float>(q[i * 32 + lane]) * a.scale_log2;
#pragma unroll
  for (int i = 0; i < VL; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = warp; j < keys.n; j += kWarps) {
    const int32_t raw = fetch_key(a, keys, j);
    const Key k = locate_key(a, keys, j, raw);
    if (bad_key(keys, j, raw, k) && lane == 0) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
    if (!k.valid) continue;
    const uint8_t* kp = a.cache.k + k.block * a.cache.k_block + k.offset * a.cache.k_token + kv * a.cache.k_head;
    const uint8_t* vp = a.cache.v + k.block * a.cache.v_block + k.offset * a.cache.v_token + kv * a.cache.v_head;
    const float ks = a.cache.k_scale[static_cast<int64_t>(k.block) * a.cache.kv_heads + kv];
    const float vs = a.cache.v_scale[static_cast<int64_t>(k.block) * a.cache.kv_heads + kv];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < KL; ++i) s += qr[i] * e4m3_to_float(kp[i * 32 + lane]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(kAllLanes, s, d);
    s *= ks;
    const float top = fmaxf(m, s);
    const float grow = m == -INFINITY ? 0.f : exp2f(m - top);
    const float p = exp2f(s - top);
    l = l * grow + p;
    m = top;
#pragma unroll
    for (int i = 0; i < VL; ++i) o[i] = o[i] * grow + p * vs * e4m3_to_float(vp[i * 32 + lane]);
  }
  if (lane == 0) {
    shared_m[warp] = m;
    shared_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < VL; ++i) shared_o[warp][i * 32 + lane] = o[i];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, shared_m[w]);
  float f[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    f[w] = shared_m[w] == -INFINITY && shared_l[w] == 0.f ? 0.f : exp2f(shared_m[w] - top);
    total += f[w] * shared_l[w];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* out = static_cast<T*>(a.out) + row * a.out_row + head * a.out_head;
  for (int d = threadIdx.x; d < DV; d += kWarps * 32) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x += f[w] * shared_o[w][d];
    out[d] = static_cast<T>(x * inv);
  }
  if (threadIdx.x == 0) {
    a.lse[static_cast<int64_t>(row) * a.heads + head] =
        total == 0.f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
  }
}

template <typename T>
int launch_typed(const AttendArgs& a, int key_dim, int64_t items, cudaStream_t stream) {
  void (*fn)(AttendArgs) = key_dim == 64 ? attend_kernel<T, 64, 64>
                           : key_dim == 128 ? attend_kernel<T, 128, 128> : attend_kernel<T, 576, 512>;
  const int64_t grid = items * a.heads;
  if (grid > 0x7fffffff) return SILKERN_E_SHAPE;
  return launch_pdl(fn, static_cast<unsigned>(grid), kWarps * 32, 0, 1, stream, a);
}

}  // namespace

int launch_attend(const AttendArgs& a, int key_dim, int type, cudaStream_t stream) {
  const int64_t items = a.slots != nullptr ? a.rows : static_cast<int64_t>(a.rows) + a.sequences;
  return type == SILKERN_BF16 ? launch_typed<__nv_bfloat16>(a, key_dim, items, stream)
                              : launch_typed<__half>(a, key_dim, items, stream);
}

}  // namespace silkern
