// chm_host.h -- host-side bookkeeping shared by the translation units of the
// library: launch accounting and the optional per-launch timing.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace chm {

// Counts one launch on this thread and turns a launch error into a chm_status.
int launch_status();

// Starts the count that chm_last_launch_count() returns.
void launches_reset();

// CUDA events around one launch of a kernel class while timing is enabled.
class ScopedLaunchTimer {
 public:
  ScopedLaunchTimer(int cls, cudaStream_t st);
  ~ScopedLaunchTimer();
  ScopedLaunchTimer(const ScopedLaunchTimer&) = delete;
  ScopedLaunchTimer& operator=(const ScopedLaunchTimer&) = delete;

 private:
  int cls_;
  cudaStream_t st_;
  cudaEvent_t start_ = nullptr, stop_ = nullptr;
};

constexpr int kTimingScore = 5;   // the "scoring" class of chm_timing_collect

}  // namespace chm
