// Attention behind shared prefixes over caches with heads of 128 columns.
#include "shared_kernel.cuh"

namespace silkern {

int launch_shared_dim128(const SharedArgs& a, bool half, unsigned grid, cudaStream_t stream) {
  return half ? shared::launch<__half, 128>(a, grid, stream) : shared::launch<__nv_bfloat16, 128>(a, grid, stream);
}

}  // namespace silkern
