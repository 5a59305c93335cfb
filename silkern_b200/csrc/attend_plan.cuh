// How one attention call is laid over the GPU, and the launchers of the
// kernel for each cache shape (one translation unit each).
#pragma once

#include "paged.cuh"

namespace silkern {

// CTAs of a thread-block cluster at most.
constexpr int kMostCluster = 16;

struct AttendPlan {
  FastDiv per;     // queries of one sequence that share a work item
  FastDiv group;   // by heads to a cache head
  int32_t blocks;  // column blocks of one (item, cache head)
  // Work items: [0, whole) go to a pipeline each, [whole, units) are split
  // over the pipelines of a cluster each.
  uint32_t whole, units;
};

struct AttendLaunch {
  int columns;  // 16, 32 or 64 (query, head) pairs to a CTA
  bool half;    // fp16 queries
  unsigned grid, cluster;
  cudaStream_t stream;
};

// How many clusters of `size` CTAs of these kernels (which all take a whole SM)
// the current device holds at once. Asked once for each device and size; 0 on
// failure.
int resident_clusters(int size);

int launch_dim64(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l);
int launch_dim128(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l);
int launch_latent(const AttendArgs& a, const AttendPlan& plan, const AttendLaunch& l);

}  // namespace silkern
