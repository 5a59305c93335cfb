// Reading the 8-bit paged cache back.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "cache_checks.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "silkern_b200.h"
#include "tcgen05.cuh"

namespace silkern {

namespace {

struct ReadArgs {
  PagedCache cache;
  void* keys;
  void* values;
  int64_t key_token, key_head, value_token, value_head;  // elements
  bool wide;  // rows of the outputs start on 16-byte boundaries
  int32_t tokens, sequences;
  const int32_t* cu_tokens;
  const int32_t* starts;
  const int32_t* req_ids;
  const int32_t* table;
  int64_t table_rows;
  uint32_t table_width;
  Ownership own;
  FastDiv heads;  // by the cache's heads
  int32_t* status;
};

constexpr int kReadThreads = 256;
constexpr int kReadRows = 32;  // positions to a CTA, a lane each

// Sequence b owns the items from (cu[b] + 31 b) / 32 on, at least one for each 32
// of its tokens, so that (tokens + 31 sequences) / 32 items cover them all.
__device__ __forceinline__ int64_t first_read_item(int32_t cu, int32_t b) {
  return (cu + int64_t{kReadRows - 1} * b) / kReadRows;
}

template <typename T>
__device__ __forceinline__ uint32_t two_codes(uint32_t codes, float scale) {
  const uint32_t h = e4m3x2_to_f16x2(static_cast<uint16_t>(codes));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f.x * scale, f.y * scale);
    return *reinterpret_cast<const uint32_t*>(&p);
  } else {
    const __half2 p = __floats2half2_rn(f.x * scale, f.y * scale);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
}

// One CTA for 32 positions of one sequence, all heads, keys and values. Each
// warp looks its CTA's positions up, a lane each (owner, page, block); then
// every thread takes 16 codes at a time: one load, two stores. The product of
// code and scale is rounded to float32 (exact for a power of two) and then to
// the output's type. Bound by memory, two thirds of it stores: 65536 tokens of 8
// heads of 128 (403 MB) 75 us, 5.35 TB/s.
template <typename T, int DIM>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ ReadArgs a) {
  constexpr uint32_t kPieces = DIM / 16;
  __shared__ int32_t row_of[kReadRows];
  __shared__ uint32_t block_of[kReadRows], offset_of[kReadRows];
  pdl_wait();
  pdl_launch_dependents();
  const int32_t lane = threadIdx.x & 31;
  const int32_t item = blockIdx.x;
  int32_t low = 0, high = a.sequences;
  while (high - low > 1) {
    const int32_t step = (high - low + 31) / 32;
    const int32_t b = low + lane * step;
    const bool before = b < high && first_read_item(min(max(load_int(a.cu_tokens + b), 0), a.tokens), b) <= item;
    const uint32_t hits = __ballot_sync(kAllLanes, before);
    const int32_t last = hits == 0 ? 0 : 31 - __clz(hits);
    low += last * step;
    high = min(high, low + step);
  }
  const int32_t begin = min(max(load_int(a.cu_tokens + low), 0), a.tokens);
  const int32_t end = min(max(load_int(a.cu_tokens + low + 1), begin), a.tokens);
  const int64_t part = item - first_read_item(begin, low);
  const int64_t first = begin + part * kReadRows;
  if (part < 0 || first >= end) return;
  const int32_t start = load_int(a.starts + low);
  const int32_t req = load_int(a.req_ids + low);
  if (start < 0 || static_cast<int64_t>(start) + (end - begin) > 0x7fffffff) {
    if (part == 0 && threadIdx.x == 0) flag_status(a.status, SILKERN_STATUS_BAD_LENGTH);
    return;
  }
  if (req < 0 || req >= a.table_rows) {
    if (part == 0 && threadIdx.x == 0) flag_status(a.status, SILKERN_STATUS_BAD_REQUEST);
    return;
  }
  // This lane's position; the owned ones come together.
  const int32_t row = static_cast<int32_t>(first) + lane;
  const uint32_t position = static_cast<uint32_t>(start) + static_cast<uint32_t>(row - begin);
  const uint32_t run = fastdiv(position, a.own.group);
  const uint32_t within = position - run * a.own.group.divisor - a.own.rank_first;  // wraps where a rank before owns it
  bool mine = row < end && within < a.own.interleave.divisor;
  uint32_t block = 0, offset = 0;
  if (mine) {
    const uint32_t local = run * a.own.interleave.divisor + within;
    const uint32_t page = fastdiv(local, a.cache.block);
    offset = local - page * a.cache.block.divisor;
    const int32_t found = page < a.table_width ? load_int(a.table + static_cast<int64_t>(req) * a.table_width + page) : -1;
    block = static_cast<uint32_t>(found);
    mine = block < a.cache.num_blocks;
    if (!mine && threadIdx.x < 32) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
  }
  const uint32_t all = __ballot_sync(kAllLanes, mine);
  if (threadIdx.x < 32 && mine) {
    const int at = __popc(all & lanemask_lt());
    row_of[at] = row;
    block_of[at] = block;
    offset_of[at] = offset;
  }
  __syncthreads();
  const uint32_t rows = __popc(all), heads = a.cache.kv_heads;
  const uint32_t each = rows * heads * kPieces;
  const bool values = a.values != nullptr;
  const uint32_t total = values ? 2 * each : each;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < total; i += kReadThreads) {
    const bool is_value = i >= each;
    const uint32_t j = is_value ? i - each : i;
    const uint32_t pair = j / kPieces, piece = j - pair * kPieces, r = fastdiv(pair, a.heads), head = pair - r * heads;
    const uint8_t* src = is_value ? a.cache.v + block_of[r] * a.cache.v_block + offset_of[r] * a.cache.v_token + head * a.cache.v_head
                                  : a.cache.k + block_of[r] * a.cache.k_block + offset_of[r] * a.cache.k_token + head * a.cache.k_head;
    const float scale = (is_value ? a.cache.v_scale : a.cache.k_scale)[static_cast<int64_t>(block_of[r]) * heads + head];
    T* dst = static_cast<T*>(is_value ? a.values : a.keys) + row_of[r] * (is_value ? a.value_token : a.key_token) +
             head * (is_value ? a.value_head : a.key_head) + piece * 16;
    const uint4 raw = *reinterpret_cast<const uint4*>(src + piece * 16);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t y[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[2 * k] = two_codes<T>(w[k] & 0xffffu, scale);
      y[2 * k + 1] = two_codes<T>(w[k] >> 16, scale);
    }
    if (a.wide) {
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(y[0], y[1], y[2], y[3]);
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(y[4], y[5], y[6], y[7]);
    } else {
      const T* e = reinterpret_cast<const T*>(y);
#pragma unroll
      for (int k = 0; k < 16; ++k) dst[k] = e[k];
    }
  }
}

template <typename T>
void (*read_for(int dim))(ReadArgs) {
  return dim == 64 ? read_kernel<T, 64> : dim == 128 ? read_kernel<T, 128> : read_kernel<T, 576>;
}

}  // namespace
}  // namespace silkern

using namespace silkern;

extern "C" int silkern_read_quantized_v1(const silkern_cache_v1* cache, void* keys, int64_t key_token, int64_t key_head,
                                         void* values, int64_t value_token, int64_t value_head, int32_t type,
                                         int64_t tokens, const int32_t* cu_tokens, const int32_t* starts,
                                         const int32_t* req_ids, int64_t sequences, const int32_t* block_table,
                                         int64_t table_rows, int64_t table_width, int32_t dcp_size, int32_t dcp_rank,
                                         int32_t dcp_interleave, int32_t* status, void* stream) {
  ReadArgs a{};
  int rc = check_cache(cache, &a.cache);
  if (rc != SILKERN_OK) return rc;
  const bool latent = cache->key_dim == 576;
  if (!keys || (!latent && !values) || !cu_tokens || !starts || !req_ids || !block_table) return SILKERN_E_NULL;
  if (latent && values != nullptr) return SILKERN_E_CACHE;
  if (type != SILKERN_BF16 && type != SILKERN_F16) return SILKERN_E_TYPE;
  if (tokens < 1 || tokens > 0x7fffffff || sequences < 1 || sequences > 0x3fffffff || table_rows < 1 || table_width < 1 ||
      table_width > 0x7fffffff) {
    return SILKERN_E_SHAPE;
  }
  rc = check_owner(cache->block_size, dcp_size, dcp_rank, dcp_interleave, &a.own);
  if (rc != SILKERN_OK) return rc;
  const Place written[2] = {
      Place(keys, 2 * int64_t{cache->key_dim}).along(tokens, 2 * key_token).along(cache->kv_heads, 2 * key_head),
      Place(values, 2 * int64_t{cache->value_dim}).along(tokens, 2 * value_token).along(cache->kv_heads, 2 * value_head)};
  const Place read[8] = {place_of_keys(cache), place_of_values(cache), place_of_scales(cache, cache->k_scale),
                         place_of_scales(cache, cache->v_scale), Place(cu_tokens, 4 * (sequences + 1)),
                         Place(starts, 4 * sequences), Place(req_ids, 4 * sequences),
                         Place(block_table, 4 * table_rows * table_width)};
  if (shares(written, read)) return SILKERN_E_ALIAS;
  a.keys = keys;
  a.values = values;
  a.key_token = key_token;
  a.key_head = key_head;
  a.value_token = value_token;
  a.value_head = value_head;
  a.wide = (key_token | key_head | value_token | value_head) % 8 == 0 &&
           (reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) % 16 == 0;
  a.tokens = static_cast<int32_t>(tokens);
  a.sequences = static_cast<int32_t>(sequences);
  a.cu_tokens = cu_tokens;
  a.starts = starts;
  a.req_ids = req_ids;
  a.table = block_table;
  a.table_rows = table_rows;
  a.table_width = static_cast<uint32_t>(table_width);
  a.heads = make_fastdiv(static_cast<uint32_t>(cache->kv_heads));
  a.status = status;
  const int64_t items = (tokens + (kReadRows - 1) * sequences) / kReadRows;
  if (items > 0x7fffffff) return SILKERN_E_SHAPE;
  void (*fn)(ReadArgs) = type == SILKERN_BF16 ? read_for<__nv_bfloat16>(cache->key_dim) : read_for<__half>(cache->key_dim);
  return launch_pdl(fn, static_cast<unsigned>(items), kReadThreads, 0, 1, static_cast<cudaStream_t>(stream), a);
}
