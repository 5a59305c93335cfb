// The attention kernel for a latent cache.
#include "attend_kernel.cuh"

namespace silkern {

int launch_latent(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  return launch_shape<kLatent>(a, plan, l);
}

}  // namespace silkern
