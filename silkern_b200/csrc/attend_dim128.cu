// The attention kernel for heads of 128.
#include "attend_kernel.cuh"

namespace silkern {

int launch_dim128(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  return launch_shape<kDim128>(a, plan, l);
}

}  // namespace silkern
