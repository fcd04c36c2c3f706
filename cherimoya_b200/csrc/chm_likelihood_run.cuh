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

// How a launch is cut: threads of a team, blocks of a row's cluster, and the
// vectors of a block's chunk (a multiple of the threads).
struct Cut {
  int threads, blocks, cap;
};

int largest(const Rows& a) { return *std::max_element(a.size, a.size + a.ng); }

// A warp takes a short row, a block of 128, 256 or 512 threads a longer one;
// rows of more than kChunkBytes are shared by the blocks of a cluster, so that
// each holds its share, and few long rows are cut further, to reach more SMs.
constexpr int kChunkBytes = 96 << 10;
Cut cut_rows(int nvec, long long rows, bool warp) {
  Cut c{};
  c.blocks = 1;
  while (c.blocks < kMaxCluster && nvec > c.blocks * (kChunkBytes / 16)) c.blocks *= 2;
  while (c.blocks < kMaxCluster && rows * c.blocks < 2 * 148 && nvec > c.blocks * 512)
    c.blocks *= 2;
  const int share = (nvec + c.blocks - 1) / c.blocks;
  c.threads = warp && share <= 64 ? 32 : share <= 1024 ? 128 : share <= 4096 ? 256 : 512;
  if (c.blocks > 1 && c.threads < 256) c.threads = 256;
  const int most = std::min(std::max(share, 1), kChunkBytes / 16);
  c.cap = (most + c.threads - 1) / c.threads * c.threads;
  return c;
}

template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), int threads, int blocks, long long rows, size_t smem,
           cudaStream_t st, bool cluster, Args... args) {
  const int per_block = threads == 32 ? 4 : 1;
  const long long grid = (rows + per_block - 1) / per_block * blocks;
  if (grid > INT_MAX) return CHM_ERR_UNSUPPORTED;
  if (smem > 32 << 10 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
          cudaSuccess)
    return CHM_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads * per_block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster && blocks > 1 ? 1 : 0;
  ScopedLaunchTimer timer(kTimingScore, st);
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return launch_status();
}

}  // namespace

template <typename T, bool kMask>
int run_log_probs_m(const Rows& a, const ScoreArgs& o, long long n, cudaStream_t st) {
  const Cut c = cut_rows(largest(a) / Vec<T>::N, n, o.top_k <= 8);
  const size_t smem = (size_t)(c.threads == 32 ? 4 : 1) * c.cap * 16 +
                      (c.blocks > 1 ? sizeof(ScoreCluster) : 0);
  auto run = [&](auto kernel) {
    return launch(kernel, c.threads, c.blocks, n, smem, st, true, a, o, (unsigned)n, c.blocks,
                  c.cap);
  };
  switch (c.threads) {
    case 32: return run(log_probs_kernel<T, 32, kMask>);
    case 128: return run(log_probs_kernel<T, 128, kMask>);
    case 256: return run(log_probs_kernel<T, 256, kMask>);
    default: return run(log_probs_kernel<T, 512, kMask>);
  }
}

template <typename T>
int run_log_probs(const Rows& a, const ScoreArgs& o, long long n, cudaStream_t st) {
  return a.mask ? run_log_probs_m<T, true>(a, o, n, st) : run_log_probs_m<T, false>(a, o, n, st);
}

template <typename T, bool kMask>
int run_log_probs_grad_m(const Rows& a, const ScoreGradArgs& o, long long n, cudaStream_t st) {
  const int nvec = largest(a) / Vec<T>::N;
  // no exchange between blocks: long rows are cut into blocks of 256 x 16 vectors
  const int threads = nvec <= 256 ? 32 : 256, blocks = threads == 32 ? 1 : (nvec + 4095) / 4096;
  const int spots = o.n_targets * (o.g_log_probs != nullptr) + o.top_k * (o.g_top != nullptr);
  const size_t smem = (size_t)(threads == 32 ? 4 : 1) * spots * 8;
  auto run = [&](auto kernel) {
    return launch(kernel, threads, blocks, n, smem, st, false, a, o, (unsigned)n, blocks);
  };
  return threads == 32 ? run(log_probs_grad_kernel<T, 32, kMask>)
                       : run(log_probs_grad_kernel<T, 256, kMask>);
}

template <typename T>
int run_log_probs_grad(const Rows& a, const ScoreGradArgs& o, long long n, cudaStream_t st) {
  return a.mask ? run_log_probs_grad_m<T, true>(a, o, n, st)
                : run_log_probs_grad_m<T, false>(a, o, n, st);
}

template <typename T, bool kMask>
int run_distill_m(const Rows& a, const DistillArgs& o, long long n, cudaStream_t st) {
  const int nvec = largest(a) / Vec<T>::N;
  const Cut c = cut_rows(nvec, n, o.n_listed <= 128);
  const int team =
      distill_bytes(o.n_listed, c.cap, (nvec + c.blocks - 1) / c.blocks, Vec<T>::N);
  const size_t smem = (size_t)(c.threads == 32 ? 4 : 1) * team;
  auto run = [&](auto kernel) {
    return launch(kernel, c.threads, c.blocks, n, smem, st, true, a, o, (unsigned)n, c.blocks,
                  c.cap, team);
  };
  switch (c.threads) {
    case 32: return run(distill_kernel<T, 32, kMask>);
    case 128: return run(distill_kernel<T, 128, kMask>);
    case 256: return run(distill_kernel<T, 256, kMask>);
    default: return run(distill_kernel<T, 512, kMask>);
  }
}

template <typename T>
int run_distill(const Rows& a, const DistillArgs& o, long long n, cudaStream_t st) {
  return a.mask ? run_distill_m<T, true>(a, o, n, st) : run_distill_m<T, false>(a, o, n, st);
}

}  // namespace lk
}  // namespace chm
