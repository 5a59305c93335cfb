// Argument checks of the entry points over the 8-bit paged cache: geometry,
// ownership, and which buffers share memory. Host only.
#pragma once

#include <cstdint>

#include "host.cuh"
#include "paged.cuh"
#include "silkern_b200.h"

namespace silkern {

// The bytes of a strided buffer: `bytes` from every place begin + i stride[0] +
// j stride[1] + ..., i below count[0] and so on, largest strides first.
struct Place {
  uintptr_t begin = 0;
  int64_t bytes = 0;
  int dims = 0;
  int64_t count[3], stride[3];

  Place(const void* base, int64_t inner) : begin(reinterpret_cast<uintptr_t>(base)), bytes(base == nullptr ? 0 : inner) {}
  Place&& along(int64_t n, int64_t step) && {
    if (n > 1) {
      if (step < 0) {  // the same places, from the lowest
        begin += static_cast<uintptr_t>((n - 1) * step);
        step = -step;
      }
      int at = dims++;
      for (; at > 0 && stride[at - 1] < step; --at) {
        count[at] = count[at - 1];
        stride[at] = stride[at - 1];
      }
      count[at] = n;
      stride[at] = step;
    }
    return static_cast<Place&&>(*this);
  }
  // From the first byte to behind the last, of the dimensions from `from` on.
  int64_t extent(int from) const {
    int64_t n = bytes;
    for (int i = from; i < dims; ++i) n += (count[i] - 1) * stride[i];
    return n;
  }
};

// Whether a's dimensions from `i` on at 0 and b's from `j` on at `shift` share
// no byte. Buffers that take turns in memory, as column slices of one tensor
// or pages of one allocation do, have their largest stride in common: what lies
// between two of its steps is then compared alone. Else by their extents.
inline bool apart(const Place& a, int i, const Place& b, int j, int64_t shift) {
  if (shift >= a.extent(i) || shift + b.extent(j) <= 0) return true;
  if (i == a.dims || j == b.dims || a.stride[i] != b.stride[j] || a.stride[i] < 1) return false;
  const int64_t step = a.stride[i];
  if (a.extent(i + 1) > step || b.extent(j + 1) > step) return false;
  const int64_t ahead = (shift % step + step) % step;
  return apart(a, i + 1, b, j + 1, ahead) && apart(a, i + 1, b, j + 1, ahead - step);
}
// Whether every step of a dimension leaves the smaller ones' extent behind.
inline bool single(const Place& a) {
  for (int i = 0; i < a.dims; ++i) {
    if (a.stride[i] < a.extent(i + 1)) return false;
  }
  return true;
}
inline bool shares(const Place& a, const Place& b) {
  return a.bytes != 0 && b.bytes != 0 &&
         !apart(a, 0, b, 0, static_cast<int64_t>(b.begin) - static_cast<int64_t>(a.begin));
}
// Whether an output shares memory with another output, an input or itself.
template <int N, int M>
bool shares(const Place (&outputs)[N], const Place (&inputs)[M]) {
  for (int i = 0; i < N; ++i) {
    if (!single(outputs[i])) return true;
    for (int j = 0; j < M; ++j) {
      if (shares(outputs[i], inputs[j])) return true;
    }
    for (int j = 0; j < i; ++j) {
      if (shares(outputs[i], outputs[j])) return true;
    }
  }
  return false;
}

inline Place place_of_keys(const silkern_cache_v1* c) {
  return Place(c->k, c->key_dim).along(c->num_blocks, c->k_block).along(c->block_size, c->k_token).along(c->kv_heads, c->k_head);
}
inline Place place_of_values(const silkern_cache_v1* c) {
  return Place(c->v, c->value_dim).along(c->num_blocks, c->v_block).along(c->block_size, c->v_token).along(c->kv_heads, c->v_head);
}
inline Place place_of_scales(const silkern_cache_v1* c, const float* scale) {
  return Place(scale, c->num_blocks * c->kv_heads * 4);
}

inline int check_cache(const silkern_cache_v1* c, PagedCache* out) {
  if (c == nullptr || c->k == nullptr || c->k_scale == nullptr) return SILKERN_E_NULL;
  const bool latent = c->key_dim == 576;
  if (!latent && (c->v == nullptr || c->v_scale == nullptr)) return SILKERN_E_NULL;
  if (latent ? (c->value_dim != 512 || c->kv_heads != 1 || c->v != nullptr || c->v_scale != nullptr)
             : ((c->key_dim != 64 && c->key_dim != 128) || c->value_dim != c->key_dim)) {
    return SILKERN_E_CACHE;
  }
  if (c->kv_heads < 1 || c->kv_heads > 65535 || c->num_blocks < 1) return SILKERN_E_CACHE;
  if (c->block_size < 1 || c->block_size > 65536) return SILKERN_E_BLOCK_SIZE;
  if (c->num_blocks > 0x7fffffff / c->block_size) return SILKERN_E_CACHE;
  const int64_t strides[6] = {c->k_block, c->k_token, c->k_head, latent ? 0 : c->v_block,
                              latent ? 0 : c->v_token, latent ? 0 : c->v_head};
  for (const int64_t s : strides) {
    if (s < 0 || s % 16 != 0) return SILKERN_E_CACHE;
  }
  if (reinterpret_cast<uintptr_t>(c->k) % 16 != 0 || reinterpret_cast<uintptr_t>(c->v) % 16 != 0) {
    return SILKERN_E_CACHE;
  }
  out->k = static_cast<const uint8_t*>(c->k);
  out->v = latent ? out->k : static_cast<const uint8_t*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = latent ? c->k_scale : c->v_scale;
  out->k_block = c->k_block;
  out->k_token = c->k_token;
  out->k_head = c->k_head;
  out->v_block = latent ? c->k_block : c->v_block;
  out->v_token = latent ? c->k_token : c->v_token;
  out->v_head = latent ? c->k_head : c->v_head;
  out->num_blocks = static_cast<uint32_t>(c->num_blocks);
  out->kv_heads = static_cast<uint32_t>(c->kv_heads);
  out->block = make_fastdiv(static_cast<uint32_t>(c->block_size));
  return SILKERN_OK;
}

inline int check_owner(int32_t block_size, int32_t dcp_size, int32_t dcp_rank, int32_t interleave, Ownership* out) {
  if (dcp_size < 1 || dcp_rank < 0 || dcp_rank >= dcp_size || interleave < 1) return SILKERN_E_DCP;
  if (static_cast<int64_t>(dcp_size) * interleave > 0x7fffffff) return SILKERN_E_DCP;
  if (block_size % interleave != 0) return SILKERN_E_BLOCK_SIZE;
  out->group = make_fastdiv(static_cast<uint32_t>(dcp_size) * static_cast<uint32_t>(interleave));
  out->interleave = make_fastdiv(static_cast<uint32_t>(interleave));
  out->rank_first = static_cast<uint32_t>(dcp_rank) * static_cast<uint32_t>(interleave);
  return SILKERN_OK;
}

}  // namespace silkern
