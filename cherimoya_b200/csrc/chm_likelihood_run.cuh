// chm_likelihood_run.cuh -- launch configurations of the likelihood and
// distillation kernels, instantiated per logits type.
#pragma once
#include <algorithm>
#include <climits>

#include "../../include/cherimoya_b200.h"
#include "chm_host.h"
#include "chm_likelihood.cuh"

namespace chm {
namespace lk {
namespace {

// How a launch is cut: threads of a team and blocks of a row's cluster.
struct Cut {
  int threads, blocks;
};

constexpr int kVecs = 8;          // 16-byte vectors that a thread holds

// Vectors of the launch's longest row, with one to spare for rows that begin
// inside a granule.
int longest(const Rows& a, int n) {
  return (*std::max_element(a.size, a.size + a.ng) + n - 1) / n + 1;
}

// A warp takes a row that it holds in registers, else a block of 128 or 256
// threads; longer rows are shared by the blocks of a cluster, so that each
// holds its share. Few long rows are cut further, to reach more SMs.
Cut cut_rows(int nvec, long long rows, bool wide) {
  if (!wide && nvec <= 32 * kVecs) return {32, 1};
  if (nvec <= 128 * kVecs) return {128, 1};
  int blocks = 1;
  while (blocks < kMaxCluster && nvec > blocks * 256 * kVecs) blocks *= 2;
  while (blocks < kMaxCluster && rows * blocks < 148 && nvec > blocks * 512) blocks *= 2;
  return {nvec > blocks * 256 * kVecs ? 512 : 256, blocks};
}

template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), const Cut& cut, long long rows, size_t smem, cudaStream_t st,
           bool cluster, Args... args) {
  const int per_block = cut.threads == 32 ? 4 : 1;
  const long long grid = (rows + per_block - 1) / per_block * cut.blocks;
  if (grid > INT_MAX) return CHM_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(cut.threads * per_block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cut.blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster && cut.blocks > 1 ? 1 : 0;
  ScopedLaunchTimer timer(kTimingScore, st);
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return launch_status();
}

}  // namespace

template <typename T>
int run_log_probs(const Rows& a, const ScoreArgs& o, long long n, cudaStream_t st) {
  const Cut cut = cut_rows(longest(a, Vec<T>::N), n, o.top_k > 32);
  auto run = [&](auto kernel) {
    return launch(kernel, cut, n, 0, st, true, a, o, (unsigned)n, cut.blocks);
  };
  switch (cut.threads) {
    case 32: return run(log_probs_kernel<T, 32, kVecs, 6>);
    case 128: return run(log_probs_kernel<T, 128, kVecs, 6>);
    case 256: return run(log_probs_kernel<T, 256, kVecs, 3>);
    default: return run(log_probs_kernel<T, 512, kVecs, 1>);
  }
}

template <typename T>
int run_log_probs_grad(const Rows& a, const ScoreGradArgs& o, long long n, cudaStream_t st) {
  const int nvec = longest(a, Vec<T>::N);
  // no exchange between blocks: long rows are cut into blocks of 256 x 4 vectors
  const Cut cut = nvec <= 32 * kVecs ? Cut{32, 1} : Cut{256, (nvec + 1023) / 1024};
  const int spots = o.n_targets * (o.g_log_probs != nullptr) + o.top_k * (o.g_top != nullptr);
  const size_t smem = (size_t)(cut.threads == 32 ? 4 : 1) * spots * 8;
  auto run = [&](auto kernel) {
    return launch(kernel, cut, n, smem, st, false, a, o, (unsigned)n, cut.blocks);
  };
  return cut.threads == 32 ? run(log_probs_grad_kernel<T, 32, kVecs>)
                           : run(log_probs_grad_kernel<T, 256, 4>);
}

template <typename T>
int run_distill(const Rows& a, const DistillArgs& o, long long n, cudaStream_t st) {
  const int nvec = longest(a, Vec<T>::N);
  const Cut cut = cut_rows(nvec, n, o.n_listed > 128);
  const int team =
      distill_bytes(o.n_listed, (nvec + cut.blocks - 1) / cut.blocks, Vec<T>::N);
  const size_t smem = (size_t)(cut.threads == 32 ? 4 : 1) * team;
  auto run = [&](auto kernel) {
    return launch(kernel, cut, n, smem, st, true, a, o, (unsigned)n, cut.blocks, team);
  };
  switch (cut.threads) {
    case 32: return run(distill_kernel<T, 32, kVecs, 5>);
    case 128: return run(distill_kernel<T, 128, kVecs, 5>);
    case 256: return run(distill_kernel<T, 256, kVecs, 3>);
    default: return run(distill_kernel<T, 512, kVecs, 1>);
  }
}

}  // namespace lk
}  // namespace chm
