// The attention kernel for heads of 64.
#include "attend_kernel.cuh"

namespace silkern {

int launch_dim64(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  return launch_shape<kDim64>(a, plan, l);
}

int resident_clusters(int size) {
  using C = Config<kDim64, 16, 2>;
  const auto kernel = attend_kernel<kDim64, 16, 2>;
  static DeviceBits granted{0};
  static std::atomic<int> known[kNotedDevices][kMostCluster + 1];  // one more than the number; 0: not asked yet
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  if (device < kNotedDevices) {
    const int told = known[device][size].load(std::memory_order_relaxed);
    if (told > 0) return told - 1;
  }
  if (allow_launch(reinterpret_cast<const void*>(kernel), kSharedMemory, granted) != SILKERN_OK) return 0;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(size, 1, 1);
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSharedMemory;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int room = 0;
  if (cudaOccupancyMaxActiveClusters(&room, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    room = 0;
  }
  if (device < kNotedDevices) known[device][size].store(room + 1, std::memory_order_relaxed);
  return room;
}

}  // namespace silkern
