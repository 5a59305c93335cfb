// The attention kernel for heads of 64.
#include <array>

#include "attend_kernel.cuh"

namespace silkern {

int launch_dim64(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l) {
  return launch_shape<kDim64>(a, plan, l);
}

int resident_clusters(int size) {
  using C = Config<kDim64, 16, 2>;
  const auto kernel = attend_kernel<kDim64, 16, 2>;
  static std::mutex mutex;
  static std::vector<std::pair<int, std::array<int, kMostCluster + 1>>> known;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || allow_launch(reinterpret_cast<const void*>(kernel), kSharedMemory) != SILKERN_OK) {
    (void)cudaGetLastError();
    return 0;
  }
  std::lock_guard<std::mutex> lock(mutex);
  for (const auto& k : known) {
    if (k.first == device) return k.second[size];
  }
  std::array<int, kMostCluster + 1> room{};
  for (int n = 1; n <= kMostCluster; ++n) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = n;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(n, 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSharedMemory;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&room[n], kernel, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      room[n] = 0;
    }
  }
  known.emplace_back(device, room);
  return room[size];
}

}  // namespace silkern
