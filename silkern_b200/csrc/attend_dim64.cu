// The attention kernel for heads of 64.
#include "attend_kernel.cuh"

namespace silkern {

int launch_dim64(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  return launch_shape<kDim64>(a, plan, l);
}

}  // namespace silkern
