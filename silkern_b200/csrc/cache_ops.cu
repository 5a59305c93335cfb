// The cache's own operators: appending tokens in 8 bits, joining the ranks'
// partial results, and the argument checks of the attention entry points.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "cache_checks.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "ptx.cuh"
#include "silkern_b200.h"

namespace silkern {

int launch_attend(AttendArgs& a, int key_dim, int type, cudaStream_t stream);

namespace {

// ---------------------------------------------------------------- append

struct AppendArgs {
  PagedCache cache;
  const void* keys;
  const void* values;
  int64_t key_token, key_head, value_token, value_head;  // elements
  bool wide;  // new values lie on 16-byte boundaries, eight by eight
  int32_t tokens, sequences;
  const int32_t* cu_tokens;
  const int32_t* starts;
  const int32_t* req_ids;
  const int32_t* table;
  int64_t table_rows;
  uint32_t table_width;
  FastDiv page_tokens;  // by block_size * dcp_size: positions from page to page
  Ownership own;
  int32_t* status;
};

// The scale that a largest magnitude asks for: the smallest power of two w
// with 448 w >= m, from the bits of m (448 = 0.875 * 2^9, so with m = f 2^e,
// f in [0.5, 1), w = 2^(e - 9), or twice that where f > 0.875).
__device__ __forceinline__ float scale_for(float m) {
  if (m == 0.f) return 0.f;
  int e;
  const float f = frexpf(m, &e);
  const int p = e - 9 + (f > 0.875f ? 1 : 0);
  return ldexpf(1.f, min(max(p, -100), 100));
}

__device__ __forceinline__ int64_t first_append_item(const AppendArgs& a, int32_t cu, int32_t b) {
  const int64_t n = cu + (2 * static_cast<int64_t>(a.page_tokens.divisor) - 2) * b;
  return n <= 0x7fffffff ? fastdiv(static_cast<uint32_t>(n), a.page_tokens) : n / a.page_tokens.divisor;
}

__device__ __forceinline__ uint8_t to_e4m3(float x) {
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float from_e4m3(uint8_t code) {
  __nv_fp8_e4m3 x;
  x.__x = code;
  return static_cast<float>(x);
}

// One CTA for each (page that a sequence's tokens touch, head, keys or
// values). Sequence b owns the items from (cu[b] + (2 p - 2) b) / p on, p the
// positions from page to page: n new tokens touch at most (n + 2 p - 2) / p
// pages of a rank. A CTA reads its new values once, 16 bytes a thread at a
// time, and keeps the first kKept of a thread's for the second pass. What
// bounds a decode step's call is its launch and the chain of dependent loads
// (item, request, page, tokens): 9 us for 64 tokens of 8 heads of 128. What
// bounds a prompt's, its few pages: 8192 tokens of a latent cache over two ranks
// are 64 of them, and take 8 us.
template <typename T, int DIM, int THREADS>
__global__ void __launch_bounds__(THREADS) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kPieces = DIM / 8;  // of 8 values in a token
  constexpr int kKept = 9;
  __shared__ uint32_t most_shared[THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t item = blockIdx.x;
  const uint32_t head = blockIdx.y;
  const bool is_value = blockIdx.z != 0;
  int32_t low = 0, high = a.sequences;
  while (high - low > 1) {
    const int32_t step = (high - low + 31) / 32;
    const int32_t b = low + lane * step;
    bool before = false;
    if (b < high) {
      const int32_t cu = min(max(load_int(a.cu_tokens + b), 0), a.tokens);
      before = first_append_item(a, cu, b) <= item;
    }
    const uint32_t hits = __ballot_sync(kAllLanes, before);
    const int32_t last = hits == 0 ? 0 : 31 - __clz(hits);
    low += last * step;
    high = min(high, low + step);
  }
  const int32_t begin = min(max(load_int(a.cu_tokens + low), 0), a.tokens);
  const int32_t end = min(max(load_int(a.cu_tokens + low + 1), begin), a.tokens);
  const int64_t page_index = item - first_append_item(a, begin, low);
  if (page_index < 0 || begin == end) return;
  const int32_t start = load_int(a.starts + low);
  const int32_t req = load_int(a.req_ids + low);
  const int64_t stop = static_cast<int64_t>(start) + (end - begin);
  if (start < 0 || stop > 0x7fffffff) {
    if (page_index == 0 && threadIdx.x == 0) flag_status(a.status, SILKERN_STATUS_BAD_LENGTH);
    return;
  }
  if (req < 0 || req >= a.table_rows) {
    if (page_index == 0 && threadIdx.x == 0) flag_status(a.status, SILKERN_STATUS_BAD_REQUEST);
    return;
  }
  // This rank's new tokens are the local tokens [first, last).
  const uint32_t first = a.own.owned_before(start), last = a.own.owned_before(static_cast<uint32_t>(stop));
  if (first == last) return;
  const uint32_t block_size = a.cache.block.divisor;
  const uint32_t page = fastdiv(first, a.cache.block) + static_cast<uint32_t>(page_index);
  const uint64_t page_first = static_cast<uint64_t>(page) * block_size;
  if (page_first >= last) return;
  const uint32_t lo = page_first > first ? static_cast<uint32_t>(page_first) : first;
  const uint32_t hi = page_first + block_size < last ? static_cast<uint32_t>(page_first) + block_size : last;
  const int32_t block = page < a.table_width ? load_int(a.table + static_cast<int64_t>(req) * a.table_width + page) : -1;
  if (static_cast<uint32_t>(block) >= a.cache.num_blocks) {
    if (threadIdx.x == 0) flag_status(a.status, SILKERN_STATUS_BAD_SLOT);
    return;
  }
  const int64_t src_token = is_value ? a.value_token : a.key_token;
  const T* src = static_cast<const T*>(is_value ? a.values : a.keys) + head * (is_value ? a.value_head : a.key_head) +
                 begin * src_token;
  const int64_t dst_token = is_value ? a.cache.v_token : a.cache.k_token;
  uint8_t* dst = const_cast<uint8_t*>(is_value ? a.cache.v : a.cache.k) +
                 block * (is_value ? a.cache.v_block : a.cache.k_block) +
                 head * (is_value ? a.cache.v_head : a.cache.k_head);
  float* scale = const_cast<float*>(is_value ? a.cache.v_scale : a.cache.k_scale) +
                 static_cast<int64_t>(block) * a.cache.kv_heads + head;
  const int32_t skip = static_cast<int32_t>(lo - page_first), count = static_cast<int32_t>(hi - lo);
  const int32_t total = count * kPieces;
  const float held_scale = *scale;
  auto read = [&](int32_t i) {
    const int32_t t = i / kPieces, d = (i - t * kPieces) * 8;
    const T* p = src + static_cast<int64_t>(a.own.position(lo + t) - static_cast<uint32_t>(start)) * src_token + d;
    uint4 x;
    if (a.wide) {
      x = *reinterpret_cast<const uint4*>(p);
    } else {
      T* e = reinterpret_cast<T*>(&x);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = p[k];
    }
    return x;
  };
  // The largest magnitude by its bits: NaN > infinity > finite.
  uint4 kept[kKept];
  uint32_t most = 0;
  auto see = [&](const uint4& x) {
    const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(static_cast<float>(e[k])) & 0x7fffffffu);
  };
#pragma unroll
  for (int n = 0; n < kKept; ++n) {
    const int32_t i = threadIdx.x + n * THREADS;
    if (i < total) kept[n] = read(i);
  }
#pragma unroll
  for (int n = 0; n < kKept; ++n) {
    if (static_cast<int32_t>(threadIdx.x) + n * THREADS < total) see(kept[n]);
  }
  for (int32_t i = threadIdx.x + kKept * THREADS; i < total; i += THREADS) see(read(i));
  most = __reduce_max_sync(kAllLanes, most);
  if (lane == 0) most_shared[warp] = most;
  __syncthreads();  // every thread has read the old scale as well
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) most = max(most, most_shared[w]);
  const bool fresh = skip == 0;
  const float old = fresh ? 0.f : held_scale;
  const float want = most >= 0x7f800000u ? NAN : scale_for(__uint_as_float(most));
  const float use = want != want || old != old ? NAN : fmaxf(old, want);
  if (threadIdx.x == 0) *scale = use;
  const bool live = use > 0.f;  // false for 0 and NaN
  // A power of two divides as its reciprocal multiplies, exactly; a scale that
  // somebody else set may be another number.
  const bool power = (__float_as_uint(use) & 0x007fffffu) == 0;
  const float inverse = __fdiv_rn(1.f, use);
  auto write = [&](int32_t i, const uint4& x) {
    const int32_t t = i / kPieces, d = (i - t * kPieces) * 8;
    const T* e = reinterpret_cast<const T*>(&x);
    uint2 codes = make_uint2(0u, 0u);
    uint8_t* c = reinterpret_cast<uint8_t*>(&codes);
    if (live) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float v = static_cast<float>(e[k]);
        c[k] = to_e4m3(power ? v * inverse : __fdiv_rn(v, use));
      }
    }
    *reinterpret_cast<uint2*>(dst + static_cast<int64_t>(skip + t) * dst_token + d) = codes;
  };
#pragma unroll
  for (int n = 0; n < kKept; ++n) {
    const int32_t i = threadIdx.x + n * THREADS;
    if (i < total) write(i, kept[n]);
  }
  for (int32_t i = threadIdx.x + kKept * THREADS; i < total; i += THREADS) write(i, read(i));
  if (!fresh && live && use > old) {  // what the page held, in the new scale
    const float ratio = __fdiv_rn(old, use);
    for (int32_t i = threadIdx.x; i < (static_cast<int32_t>(block_size) - count) * (DIM / 16); i += THREADS) {
      int32_t t = i / (DIM / 16);
      const int32_t d = (i - t * (DIM / 16)) * 16;
      if (t >= skip) t += count;
      uint4* p = reinterpret_cast<uint4*>(dst + static_cast<int64_t>(t) * dst_token + d);
      uint4 x = *p;
      uint8_t* c = reinterpret_cast<uint8_t*>(&x);
#pragma unroll
      for (int k = 0; k < 16; ++k) c[k] = to_e4m3(from_e4m3(c[k]) * ratio);
      *p = x;
    }
  }
}

template <typename T, int DIM>
void (*append_for(bool pages))(AppendArgs) {
  return pages ? append_kernel<T, DIM, 512> : append_kernel<T, DIM, 128>;
}
template <typename T>
void (*append_for(int dim, bool pages))(AppendArgs) {
  return dim == 64 ? append_for<T, 64>(pages) : dim == 128 ? append_for<T, 128>(pages) : append_for<T, 576>(pages);
}

// ---------------------------------------------------------------- merge

struct MergeArgs {
  const void* outs;
  const float* lses;
  void* out;
  float* lse;
  int64_t outs_rank, outs_row, outs_head, out_row, out_head;
  int64_t pairs;  // rows * heads
  int32_t ranks, heads, dim;
};

constexpr int kMergeWarps = 8;

// One warp for each (row, head): lane r has rank r's weight, and every lane
// eight columns at a time of all ranks, four loads on their way at once. Each
// byte is read and written once; a warp's loads of partial outputs wait for its
// lses, and for those of the columns before (8 ranks, 128 rows of 128 heads of
// 512: 152 MB in 33.5 us, 4.5 TB/s).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const __grid_constant__ MergeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5);
  if (pair >= a.pairs) return;
  const int64_t row = pair / a.heads;
  const int64_t head = pair - row * a.heads;
  const float mine = lane < a.ranks ? a.lses[lane * a.pairs + pair] : -INFINITY;
  float top = mine;
  for (int i = 32 + lane; i < a.ranks; i += 32) top = fmaxf(top, a.lses[i * a.pairs + pair]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kAllLanes, top, d));
  const float base = top == -INFINITY ? 0.f : top;
  const float weight = expf(mine - base);
  float total = 0.f;
  for (int i = 0; i < min(a.ranks, 32); ++i) total += __shfl_sync(kAllLanes, weight, i);
  for (int i = 32; i < a.ranks; ++i) total += expf(a.lses[i * a.pairs + pair] - base);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const T* src = static_cast<const T*>(a.outs) + row * a.outs_row + head * a.outs_head;
  T* dst = static_cast<T*>(a.out) + row * a.out_row + head * a.out_head;
  // The weight of rank i; 0 and `read` false where its lse is -inf.
  auto weight_of = [&](int i, bool& read) {
    const float l = i < 32 ? __shfl_sync(kAllLanes, mine, i & 31) : a.lses[i * a.pairs + pair];
    const float w = i < 32 ? __shfl_sync(kAllLanes, weight, i & 31) : expf(l - base);
    read = l != -INFINITY;
    return read ? w * inv : 0.f;
  };
  constexpr int kStep = WIDE ? 256 : 32;
  for (int d0 = 0; d0 < a.dim; d0 += kStep) {
    if constexpr (WIDE) {
      const int d = d0 + lane * 8;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int i0 = 0; i0 < a.ranks; i0 += 4) {
        uint4 raw[4];
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          raw[k] = make_uint4(0u, 0u, 0u, 0u);
          w[k] = 0.f;
          if (i0 + k < a.ranks) {
            bool read;
            w[k] = weight_of(i0 + k, read);
            if (read && d < a.dim) raw[k] = __ldcs(reinterpret_cast<const uint4*>(src + (i0 + k) * a.outs_rank + d));
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const T* v = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fmaf(w[k], static_cast<float>(v[e]), x[e]);
        }
      }
      if (d < a.dim) {
        uint4 packed;
        T* v = reinterpret_cast<T*>(&packed);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = static_cast<T>(x[e]);
        *reinterpret_cast<uint4*>(dst + d) = packed;
      }
    } else {
      const int d = d0 + lane;
      float x = 0.f;
      for (int i = 0; i < a.ranks; ++i) {
        bool read;
        const float w = weight_of(i, read);
        if (read && d < a.dim) x = fmaf(w, static_cast<float>(src[i * a.outs_rank + d]), x);
      }
      if (d < a.dim) dst[d] = static_cast<T>(x);
    }
  }
  if (a.lse != nullptr && lane == 0) a.lse[pair] = top + logf(total);
}

// ---------------------------------------------------------------- checks

// The results of an attention call share no memory with each other, with the
// cache or the queries, nor with `index`, the call's other buffers.
template <int N>
bool results_alone(const silkern_cache_v1* c, const AttendArgs& a, const Place (&index)[N]) {
  const int64_t rows = a.rows, heads = a.heads;
  const Place results[2] = {Place(a.out, 2 * c->value_dim).along(rows, 2 * a.out_row).along(heads, 2 * a.out_head),
                            Place(a.lse, 4 * rows * heads)};
  const Place read[5] = {Place(a.q, 2 * c->key_dim).along(rows, 2 * a.q_row).along(heads, 2 * a.q_head),
                         place_of_keys(c), place_of_values(c), place_of_scales(c, c->k_scale),
                         place_of_scales(c, c->v_scale)};
  return !shares(results, read) && !shares(results, index);
}

int check_queries(const silkern_cache_v1* c, const void* q, int64_t q_row, int64_t q_head, int32_t type,
                  int64_t rows, int32_t heads, void* out, int64_t out_row, int64_t out_head, float* lse,
                  float softmax_scale, AttendArgs* a) {
  if (q == nullptr || out == nullptr || lse == nullptr) return SILKERN_E_NULL;
  if (type != SILKERN_BF16 && type != SILKERN_F16) return SILKERN_E_TYPE;
  if (rows < 1 || rows > 0x7fffffff) return SILKERN_E_SHAPE;
  if (heads < 1 || heads > 65535 || heads % c->kv_heads != 0) return SILKERN_E_HEADS;
  if (q_row % 8 != 0 || q_head % 8 != 0 || reinterpret_cast<uintptr_t>(q) % 16 != 0) return SILKERN_E_CACHE;
  a->scale_log2 = softmax_scale * 1.4426950408889634f;
  if (!std::isfinite(a->scale_log2)) return SILKERN_E_ATTEND;
  a->q = q;
  a->q_row = q_row;
  a->q_head = q_head;
  a->out = out;
  a->out_row = out_row;
  a->out_head = out_head;
  a->out_wide = out_row % 8 == 0 && out_head % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  a->lse = lse;
  a->rows = static_cast<int32_t>(rows);
  a->heads = heads;
  a->heads_per_kv = heads / c->kv_heads;
  return SILKERN_OK;
}

}  // namespace
}  // namespace silkern

using namespace silkern;

extern "C" int silkern_append_quantized_v1(const silkern_cache_v1* cache, const void* keys, int64_t key_token,
                                           int64_t key_head, const void* values, int64_t value_token,
                                           int64_t value_head, int32_t type, int64_t tokens,
                                           const int32_t* cu_tokens, const int32_t* starts,
                                           const int32_t* req_ids, int64_t sequences,
                                           const int32_t* block_table, int64_t table_rows,
                                           int64_t table_width, int32_t dcp_size, int32_t dcp_rank,
                                           int32_t dcp_interleave, int32_t* status, void* stream) {
  AppendArgs a{};
  int rc = check_cache(cache, &a.cache);
  if (rc != SILKERN_OK) return rc;
  const bool latent = cache->key_dim == 576;
  if (!keys || (!latent && !values) || !cu_tokens || !starts || !req_ids || !block_table) return SILKERN_E_NULL;
  if (latent && values != nullptr) return SILKERN_E_CACHE;
  if (type != SILKERN_BF16 && type != SILKERN_F16) return SILKERN_E_TYPE;
  if (tokens < 1 || tokens > 0x7fffffff || sequences < 1 || sequences > 0x3fffffff || table_rows < 1 ||
      table_width < 1 || table_width > 0x7fffffff) {
    return SILKERN_E_SHAPE;
  }
  rc = check_owner(cache->block_size, dcp_size, dcp_rank, dcp_interleave, &a.own);
  if (rc != SILKERN_OK) return rc;
  const Place written[3] = {place_of_scales(cache, cache->k_scale), place_of_scales(cache, cache->v_scale),
                            place_of_keys(cache)};
  const Place read[6] = {Place(keys, 2 * cache->key_dim).along(tokens, 2 * key_token).along(cache->kv_heads, 2 * key_head),
                         Place(values, 2 * cache->value_dim).along(tokens, 2 * value_token).along(cache->kv_heads, 2 * value_head),
                         Place(cu_tokens, 4 * (sequences + 1)), Place(starts, 4 * sequences),
                         Place(req_ids, 4 * sequences), Place(block_table, 4 * table_rows * table_width)};
  // Keys and values may lie in one buffer, page by page or row by row.
  const Place values_too[1] = {place_of_values(cache)};
  if (shares(written, read) || shares(values_too, read) || shares(values_too, written)) return SILKERN_E_ALIAS;
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
  const int64_t page_tokens = static_cast<int64_t>(cache->block_size) * dcp_size;
  a.page_tokens = make_fastdiv(static_cast<uint32_t>(page_tokens > 0x7fffffff ? 0x7fffffff : page_tokens));
  a.status = status;
  const int64_t step = a.page_tokens.divisor;
  const int64_t items = (tokens + (2 * step - 2) * sequences) / step;
  if (items > 0x7fffffff) return SILKERN_E_SHAPE;
  // A few tokens to a sequence: small CTAs. (Half a page of the widest cache
  // fills the large ones.)
  const bool pages = tokens > 8 * sequences;
  void (*fn)(AppendArgs) = type == SILKERN_BF16 ? append_for<__nv_bfloat16>(cache->key_dim, pages)
                                                : append_for<__half>(cache->key_dim, pages);
  return launch_pdl_grid(fn, dim3(static_cast<unsigned>(items), static_cast<unsigned>(cache->kv_heads), latent ? 1 : 2),
                         pages ? 512 : 128, 0, 1, static_cast<cudaStream_t>(stream), a);
}

extern "C" int silkern_attend_selected_v1(const silkern_cache_v1* cache, const void* q, int64_t q_row, int64_t q_head,
                                          int32_t type, int64_t rows, int32_t heads, const int32_t* slots,
                                          int64_t slots_row, int64_t width, const int32_t* counts, void* out,
                                          int64_t out_row, int64_t out_head, float* lse, float softmax_scale,
                                          int32_t* status, void* stream) {
  AttendArgs a{};
  int rc = check_cache(cache, &a.cache);
  if (rc != SILKERN_OK) return rc;
  if (slots == nullptr) return SILKERN_E_NULL;
  rc = check_queries(cache, q, q_row, q_head, type, rows, heads, out, out_row, out_head, lse, softmax_scale, &a);
  if (rc != SILKERN_OK) return rc;
  if (width < 1 || width > 0x7fffffff - 4096) return SILKERN_E_SHAPE;
  a.slots = slots;
  a.slots_row = slots_row;
  a.width = static_cast<int32_t>(width);
  a.counts = counts;
  a.total_slots = static_cast<uint32_t>(cache->num_blocks * cache->block_size);
  a.status = status;
  const Place index[2] = {Place(slots, 4 * width).along(rows, 4 * slots_row), Place(counts, 4 * rows)};
  if (!results_alone(cache, a, index)) return SILKERN_E_ALIAS;
  return launch_attend(a, cache->key_dim, type, static_cast<cudaStream_t>(stream));
}

extern "C" int silkern_attend_window_v1(const silkern_cache_v1* cache, const void* q, int64_t q_row, int64_t q_head,
                                        int32_t type, int64_t rows, int32_t heads, const int32_t* cu_tokens,
                                        const int32_t* lengths, const int32_t* req_ids, int64_t sequences,
                                        const int32_t* block_table, int64_t table_rows, int64_t table_width,
                                        int64_t window, int64_t sinks, int32_t dcp_size, int32_t dcp_rank,
                                        int32_t dcp_interleave, void* out, int64_t out_row, int64_t out_head,
                                        float* lse, float softmax_scale, int32_t* status, void* stream) {
  AttendArgs a{};
  int rc = check_cache(cache, &a.cache);
  if (rc != SILKERN_OK) return rc;
  if (!cu_tokens || !lengths || !req_ids || !block_table) return SILKERN_E_NULL;
  rc = check_queries(cache, q, q_row, q_head, type, rows, heads, out, out_row, out_head, lse, softmax_scale, &a);
  if (rc != SILKERN_OK) return rc;
  if (sequences < 1 || rows + 64 * sequences > 0x7fffffff || table_rows < 1 || table_width < 1 ||
      table_width > 0x7fffffff) {
    return SILKERN_E_SHAPE;
  }
  if (window < 0 || window > 0x7fffffff || sinks < 0 || sinks > 0x7fffffff) return SILKERN_E_ATTEND;
  rc = check_owner(cache->block_size, dcp_size, dcp_rank, dcp_interleave, &a.own);
  if (rc != SILKERN_OK) return rc;
  a.cu_tokens = cu_tokens;
  a.lengths = lengths;
  a.req_ids = req_ids;
  a.sequences = static_cast<int32_t>(sequences);
  a.table = block_table;
  a.table_rows = table_rows;
  a.table_width = static_cast<uint32_t>(table_width);
  a.window = static_cast<uint32_t>(window);
  a.sinks = static_cast<uint32_t>(sinks);
  a.status = status;
  const Place index[4] = {Place(cu_tokens, 4 * (sequences + 1)), Place(lengths, 4 * sequences),
                          Place(req_ids, 4 * sequences), Place(block_table, 4 * table_rows * table_width)};
  if (!results_alone(cache, a, index)) return SILKERN_E_ALIAS;
  return launch_attend(a, cache->key_dim, type, static_cast<cudaStream_t>(stream));
}

extern "C" int silkern_merge_partials_v1(const void* outs, int64_t outs_rank, int64_t outs_row, int64_t outs_head,
                                         const float* lses, int32_t type, int64_t ranks, int64_t rows, int64_t heads,
                                         int64_t dim, void* out, int64_t out_row, int64_t out_head, float* lse,
                                         void* stream) {
  if (outs == nullptr || lses == nullptr || out == nullptr) return SILKERN_E_NULL;
  if (type != SILKERN_BF16 && type != SILKERN_F16) return SILKERN_E_TYPE;
  // (The kernel's column numbers step past dim by up to 255.)
  if (ranks < 1 || ranks > 0x7fffffff || rows < 1 || heads < 1 || heads > 0x7fffffff || dim < 1 ||
      dim > 0x7fffffff - 255 || rows > (int64_t{1} << 31) * kMergeWarps / heads - kMergeWarps) {
    return SILKERN_E_SHAPE;
  }
  MergeArgs a{outs, lses, out, lse, outs_rank, outs_row, outs_head, out_row, out_head, rows * heads,
              static_cast<int32_t>(ranks), static_cast<int32_t>(heads), static_cast<int32_t>(dim)};
  const Place written[2] = {Place(out, 2 * dim).along(rows, 2 * out_row).along(heads, 2 * out_head),
                            Place(lse, 4 * rows * heads)};
  const Place read[2] = {Place(outs, 2 * dim).along(ranks, 2 * outs_rank).along(rows, 2 * outs_row).along(heads, 2 * outs_head),
                         Place(lses, 4 * ranks * rows * heads)};
  if (shares(written, read)) return SILKERN_E_ALIAS;
  // 16 bytes at a time where every row of columns allows it.
  const bool wide = (dim | outs_rank | outs_row | outs_head | out_row | out_head) % 8 == 0 &&
                    (reinterpret_cast<uintptr_t>(outs) | reinterpret_cast<uintptr_t>(out)) % 16 == 0;
  void (*fn)(MergeArgs) = type == SILKERN_BF16 ? (wide ? merge_kernel<__nv_bfloat16, true> : merge_kernel<__nv_bfloat16, false>)
                                               : (wide ? merge_kernel<__half, true> : merge_kernel<__half, false>);
  const int64_t ctas = (a.pairs + kMergeWarps - 1) / kMergeWarps;
  if (ctas > 0x7fffffff) return SILKERN_E_SHAPE;
  return launch_pdl(fn, static_cast<unsigned>(ctas), kMergeWarps * 32, 0, 1, static_cast<cudaStream_t>(stream), a);
}
