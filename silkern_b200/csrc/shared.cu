// Attention of sequences in groups that share their first tokens.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "cache_checks.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "silkern_b200.h"
#include "tcgen05.cuh"

namespace silkern {

namespace {

struct SharedArgs {
  PagedCache cache;
  const void* q;
  int64_t q_row, q_head;
  void* out;
  int64_t out_row, out_head;
  float* lse;
  int32_t* status;
  float scale;
  int32_t rows, heads, heads_per_kv;
  int32_t sequences, groups;
  const int32_t* cu_tokens;
  const int32_t* lengths;
  const int32_t* req_ids;
  const int32_t* cu_groups;
  const int32_t* prefixes;
  const int32_t* table;
  int64_t table_rows;
  uint32_t table_width;
  Ownership own;
};

// The last i in [0, n) with at(i) <= x, for at ascending from at(0) <= x.
template <typename F>
__device__ __forceinline__ int32_t last_at_most(int32_t n, int32_t x, F at) {
  int32_t low = 0, high = n;
  while (high - low > 1) {
    const int32_t mid = low + (high - low) / 2;
    if (at(mid) <= x) low = mid; else high = mid;
  }
  return low;
}

// A warp for each (query, head), one key at a time: right for every case.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) shared_simple_kernel(const __grid_constant__ SharedArgs a) {
  constexpr int kEach = DIM / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int32_t lane = threadIdx.x & 31;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (pair >= static_cast<int64_t>(a.rows) * a.heads) return;
  const int32_t token = static_cast<int32_t>(pair / a.heads), head = static_cast<int32_t>(pair - static_cast<int64_t>(token) * a.heads);
  if (token < load_int(a.cu_tokens) || token >= load_int(a.cu_tokens + a.sequences)) return;
  const int32_t seq = last_at_most(a.sequences, token, [&](int32_t i) { return load_int(a.cu_tokens + i); });
  const int32_t position = load_int(a.lengths + seq) - (load_int(a.cu_tokens + seq + 1) - token);
  if (lane == 0 && load_int(a.lengths + seq) < load_int(a.cu_tokens + seq + 1) - load_int(a.cu_tokens + seq)) {
    flag_status(a.status, SILKERN_STATUS_BAD_LENGTH);
  }
  int32_t prefix = 0, leader = seq;
  if (seq >= load_int(a.cu_groups) && seq < load_int(a.cu_groups + a.groups)) {
    const int32_t group = last_at_most(a.groups, seq, [&](int32_t i) { return load_int(a.cu_groups + i); });
    leader = load_int(a.cu_groups + group);
    prefix = max(load_int(a.prefixes + group), 0);
  }
  const uint32_t kv = head / a.heads_per_kv;
  const T* q = static_cast<const T*>(a.q) + token * a.q_row + head * a.q_head;
  float x[kEach], y[kEach], top = -INFINITY, total = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    x[i] = static_cast<float>(q[lane * kEach + i]);
    y[i] = 0.f;
  }
  const uint32_t seen = position < 0 ? 0u : a.own.owned_before(static_cast<uint32_t>(position) + 1u);
  const uint32_t cut = a.own.owned_before(static_cast<uint32_t>(prefix));
  for (uint32_t j = 0; j < seen; ++j) {
    const int32_t req = load_int(a.req_ids + (j < cut ? leader : seq));
    if (req < 0 || req >= a.table_rows) {
      if (lane == 0) flag_status(a.status, SILKERN_STATUS_BAD_REQUEST);
      continue;
    }
    const uint32_t page = fastdiv(j, a.cache.block), offset = j - page * a.cache.block.divisor;
    const int32_t block = page < a.table_width ? load_int(a.table + req * static_cast<int64_t>(a.table_width) + page) : -1;
    if (static_cast<uint32_t>(block) >= a.cache.num_blocks) {
      if (lane == 0) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
      continue;
    }
    auto code = [](uint8_t c) {
      const uint32_t h = e4m3x2_to_f16x2(c);
      return __half2float(__low2half(*reinterpret_cast<const __half2*>(&h)));
    };
    const uint8_t* k = a.cache.k + block * a.cache.k_block + offset * a.cache.k_token + kv * a.cache.k_head;
    const uint8_t* v = a.cache.v + block * a.cache.v_block + offset * a.cache.v_token + kv * a.cache.v_head;
    const int64_t scales = static_cast<int64_t>(block) * a.cache.kv_heads + kv;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) s = fmaf(x[i], code(k[lane * kEach + i]), s);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(kAllLanes, s, d);
    s *= a.cache.k_scale[scales] * a.scale;
    const float best = fmaxf(top, s), keep = expf(top - best), weight = expf(s - best);
    top = best;
    total = total * keep + weight;
    const float w = weight * a.cache.v_scale[scales];
#pragma unroll
    for (int i = 0; i < kEach; ++i) y[i] = y[i] * keep + w * code(v[lane * kEach + i]);
  }
  T* out = static_cast<T*>(a.out) + token * a.out_row + head * a.out_head;
  const float inverse = seen == 0 || total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) out[lane * kEach + i] = static_cast<T>(y[i] * inverse);
  if (lane == 0) a.lse[pair] = top + logf(total);
}

}  // namespace
}  // namespace silkern

using namespace silkern;

extern "C" int64_t silkern_shared_workspace_v1(int64_t rows, int32_t heads, int32_t kv_heads, int32_t dim, int64_t sequences,
                                               int64_t groups) {
  if (rows < 1 || rows > 0x7fffffff || sequences < 1 || sequences > 0x3fffffff || groups < 1 || groups > 0x3fffffff) return -SILKERN_E_SHAPE;
  if (heads < 1 || heads > 65535 || kv_heads < 1 || heads % kv_heads != 0) return -SILKERN_E_HEADS;
  if (dim != 64 && dim != 128) return -SILKERN_E_CACHE;
  return 16;
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
  const int64_t needed = silkern_shared_workspace_v1(rows, heads, cache->kv_heads, cache->key_dim, sequences, groups);
  if (needed < 0) return static_cast<int>(-needed);
  if (table_rows < 1 || table_width < 1 || table_width > 0x7fffffff) return SILKERN_E_SHAPE;
  if (workspace_bytes < needed) return SILKERN_E_SCRATCH;
  if (q_row % 8 != 0 || q_head % 8 != 0 || reinterpret_cast<uintptr_t>(q) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return SILKERN_E_CACHE;
  }
  if (!std::isfinite(softmax_scale * 1.4426950408889634f)) return SILKERN_E_ATTEND;
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
  a.scale = softmax_scale;
  a.rows = static_cast<int32_t>(rows);
  a.heads = heads;
  a.heads_per_kv = heads / cache->kv_heads;
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
  const int64_t ctas = (rows * heads + 7) / 8;
  if (ctas > 0x7fffffff) return SILKERN_E_SHAPE;
  void (*fn)(SharedArgs) = type == SILKERN_BF16 ? (cache->key_dim == 64 ? shared_simple_kernel<__nv_bfloat16, 64> : shared_simple_kernel<__nv_bfloat16, 128>)
                                                : (cache->key_dim == 64 ? shared_simple_kernel<__half, 64> : shared_simple_kernel<__half, 128>);
  return launch_pdl(fn, static_cast<unsigned>(ctas), 256, 0, 1, static_cast<cudaStream_t>(stream), a);
}
