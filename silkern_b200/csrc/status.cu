// Texts of the return codes. They stand apart from the kernels' sources: a
// capture of a kernel's traffic is tied to its source, and a new code's text is
// no new kernel.
#include <cuda_runtime.h>

#include "silkern_b200.h"

extern "C" const char* silkern_status_string_v1(int code) {
  switch (code) {
    case SILKERN_OK: return "ok";
    case SILKERN_E_NULL: return "a required buffer pointer is NULL";
    case SILKERN_E_SHAPE: return "batch, width or block-table dimensions are out of range";
    case SILKERN_E_DCP: return "invalid dcp configuration";
    case SILKERN_E_BLOCK_SIZE: return "block_size must be a positive integer divisible by dcp_interleave";
    case SILKERN_E_TILE: return "unsupported tile_size";
    case SILKERN_E_ALIAS: return "an output buffer overlaps an input, another output or itself";
    case SILKERN_E_GEOMETRY: return "explicit launch geometry rejected";
    case SILKERN_E_SCRATCH:
      return "batch x tiles exceeds the allocation-free entry point's static workspace";
    case SILKERN_E_CACHE: return "unsupported cache geometry, stride or alignment";
    case SILKERN_E_HEADS: return "heads must be a positive multiple of the cache's heads";
    case SILKERN_E_TYPE: return "element type must be bfloat16 or float16";
    case SILKERN_E_ATTEND: return "window, sinks or softmax scale out of range";
    default: break;
  }
  if (code < 0) return cudaGetErrorString(static_cast<cudaError_t>(-code));
  return "unknown status";
}
