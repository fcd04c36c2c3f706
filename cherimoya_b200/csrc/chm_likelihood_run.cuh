// chm_likelihood_run.cuh -- launch configurations of the likelihood and
// distillation kernels, instantiated per logits type.
#pragma once
#include <algorithm>
#include <climits>
#include <vector>

#include "../../include/cherimoya_b200.h"
#include "chm_host.h"
#include "chm_likelihood.cuh"

namespace chm {
namespace lk {
namespace {

// How a launch is cut: threads of a team, blocks of a row's cluster (a power
// of two), and the vectors of a block's chunk (a multiple of kBatch times the threads).
struct Cut {
  int threads, log_blocks, cap;
};

int largest(const Rows& a) { return *std::max_element(a.size, a.size + a.ng); }

// Distillation with a gradient keeps a block's share of a row in shared memory
// from the first look to the last, so the row's size sets how many blocks an
// SM holds. A warp takes a short row and a block of 128 one of up to 44 KB, of
// which five fit: 8,192 x 20,000 bf16 entries take 151 us with it and 185 with
// 256 threads, 8,192 x 9,000 take 92 and 150. Above that it is a block of 256:
// 8,192 x 32,768 entries, of which three rows fit, take 220 us, 267 with 128
// threads and 326 with 512; 2,048 x 40,000, of which two fit, 101 and with 512
// 155. Rows of more than kChunkBytes are shared by the blocks of a cluster, so
// that each holds its share; few long rows are cut further, to reach more SMs.
// Many rows are not (8,192 x 32,768 in clusters of two: 387 us).
constexpr int kChunkBytes = 96 << 10;
Cut cut_rows(int nvec, long long rows, bool warp) {
  Cut c{};
  while (c.log_blocks < 3 && nvec > (kChunkBytes / 16) << c.log_blocks) ++c.log_blocks;
  while (c.log_blocks < 3 && rows << c.log_blocks < 2 * 148 && nvec > 512 << c.log_blocks)
    ++c.log_blocks;
  const int share = (nvec + (1 << c.log_blocks) - 1) >> c.log_blocks;
  c.threads = warp && share <= 256 ? 32 : share <= 2816 ? 128 : 256;
  if (c.log_blocks && c.threads < 128) c.threads = 128;
  const int most = std::min(std::max(share, 1), kChunkBytes / 16);
  c.cap = (most + kBatch * c.threads - 1) / (kBatch * c.threads) * (kBatch * c.threads);
  return c;
}

// The log probabilities read a row once, through a ring of fixed size. A warp
// takes up to 16 vectors a lane: 2,048 examples of five groups of 1,000 and 2,000
// masked fp32 entries take 50 us, 56 with teams of 64 and 79 with 128. Longer rows get
// a block of 128 (4,096 x 50,001 bf16: 88 us, 109 with 256), more than 64 top
// entries too: near as many as a warp's 128 maxima, they are bounded so loosely that most of the
// row is a candidate (10,240 x 1,000 with 128 of them 156 us, a warp per row 381; with 65
// it is 84 and 52). Few long rows are shared by the blocks of a cluster, and so are rows of which
// a thread would add up more than kMaxBatches batches one by one.
Cut cut_stream(int nvec, long long rows, int top_k) {
  Cut c{};
  c.threads = nvec <= 512 && top_k <= 64 ? 32 : 128;
  if (c.threads == 128)
    while (c.log_blocks < 3 &&
           ((rows << c.log_blocks < 6 * 148 && nvec > 1024 << c.log_blocks) ||
            nvec > kMaxBatches * kBatch * 128 << c.log_blocks))
      ++c.log_blocks;
  return c;
}

// Lets a kernel use all the dynamic shared memory that the current device has
// for a block; asked once per kernel, device and thread.
int lift_smem_limit(const void* kernel) {
  struct Known {
    const void* kernel;
    int device;
  };
  thread_local std::vector<Known> known;
  int device = 0, limit = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return CHM_ERR_CUDA;
  for (const Known& k : known)
    if (k.kernel == kernel && k.device == device) return CHM_OK;
  cudaFuncAttributes attr;
  if (cudaDeviceGetAttribute(&limit, cudaDevAttrMaxSharedMemoryPerBlockOptin, device) !=
          cudaSuccess ||
      cudaFuncGetAttributes(&attr, kernel) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           limit - (int)attr.sharedSizeBytes) != cudaSuccess)
    return CHM_ERR_CUDA;
  known.push_back({kernel, device});
  return CHM_OK;
}

// Launches a kernel with a team, or a cluster of blocks, for each row.
template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), int threads, int log_blocks, long long rows, size_t smem,
           cudaStream_t st, bool cluster, Args... args) {
  const int per_block = threads == 32 ? 4 : 1, blocks = 1 << log_blocks;
  const long long grid = (rows + per_block - 1) / per_block * blocks;
  if (grid > INT_MAX) return CHM_ERR_UNSUPPORTED;
  if (smem > 16 << 10) {
    const int status = lift_smem_limit(reinterpret_cast<const void*>(kernel));
    if (status != CHM_OK) return status;
  }
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
  const Cut c = cut_stream(largest(a) / Vec<T>::N, n, o.top_k);
  const size_t smem = (size_t)kSlots * 128 * 16 + (c.log_blocks ? sizeof(ScoreCluster) : 0);
  auto run = [&](auto kernel) {
    return launch(kernel, c.threads, c.log_blocks, n, smem, st, true, a, o, (unsigned)n,
                  c.log_blocks);
  };
  return c.threads == 32 ? run(log_probs_kernel<T, 32, kMask>)
                         : run(log_probs_kernel<T, 128, kMask>);
}

template <typename T>
int run_log_probs(const Rows& a, const ScoreArgs& o, long long n, cudaStream_t st) {
  return a.mask ? run_log_probs_m<T, true>(a, o, n, st) : run_log_probs_m<T, false>(a, o, n, st);
}

template <typename T, bool kMask>
int run_log_probs_grad_m(const Rows& a, const ScoreGradArgs& o, long long n, cudaStream_t st) {
  const int nvec = largest(a) / Vec<T>::N;
  // Nothing passes between blocks, so long rows are cut into blocks of at most 16 vectors
  // a thread: 4,096 x 8,192 bf16 entries with their forward pass take 44 us, 51 with 256 threads.
  const int threads = nvec <= 256 ? 32 : 128;
  int log_blocks = 0;
  while (threads == 128 && nvec > 2048 << log_blocks) ++log_blocks;
  const int spots = o.n_targets * (o.g_log_probs != nullptr) + o.top_k * (o.g_top != nullptr);
  const size_t smem = (size_t)(threads == 32 ? 4 : 1) * (sort_size(spots) + spots) * 4;
  auto run = [&](auto kernel) {
    return launch(kernel, threads, log_blocks, n, smem, st, false, a, o, (unsigned)n,
                  log_blocks);
  };
  return threads == 32 ? run(log_probs_grad_kernel<T, 32, kMask>)
                       : run(log_probs_grad_kernel<T, 128, kMask>);
}

template <typename T>
int run_log_probs_grad(const Rows& a, const ScoreGradArgs& o, long long n, cudaStream_t st) {
  return a.mask ? run_log_probs_grad_m<T, true>(a, o, n, st)
                : run_log_probs_grad_m<T, false>(a, o, n, st);
}

template <typename T, bool kMask>
int run_distill_m(const Rows& a, const DistillArgs& o, long long n, cudaStream_t st) {
  const int nvec = largest(a) / Vec<T>::N;
  Cut c = cut_rows(nvec, n, o.n_listed <= 128);
  int chunks = 1;
  if (!a.grad && nvec > 1024) {
    // Without a gradient nothing is looked at twice, so a block of 128 takes
    // chunks of 8 KB, the next on its way while it sums one, and seven blocks fit
    // an SM: 1,024 x 100,003 fp32 entries take 85 us (16 KB: 95; 32 KB and 256
    // threads: 96), 2,048 x 100,003 bf16 93 (103; 118), 4,096 x 25,000 fp32 83
    // (84; 104), 8,192 x 12,000 bf16 79 (held whole: 120); 500 x 100,003 fp32 lose (54 to 57,
    // 50 with 16 KB). Below 16 KB a row is one chunk. Few rows are cut until there are three
    // blocks to an SM; up to seven gave 500 x 100,003 50 but 250 x 100,003 38 instead of 35.
    c = {128, 0, 512};
    while (c.log_blocks < 3 && n << c.log_blocks < 3 * 148 && nvec >> c.log_blocks > 2048)
      ++c.log_blocks;
    chunks = 2;
  }
  const int team = distill_bytes(o.n_listed, c.cap, chunks, largest(a));
  const size_t smem = (size_t)(c.threads == 32 ? 4 : 1) * team;
  auto run = [&](auto kernel) {
    return launch(kernel, c.threads, c.log_blocks, n, smem, st, true, a, o, (unsigned)n,
                  c.log_blocks, c.cap, chunks, team);
  };
  // a chunk is a batch per thread
  const bool many = chunks > 1 && nvec > kMaxBatches * c.cap << c.log_blocks;
  switch (c.threads) {
    case 32: return run(distill_kernel<T, 32, kMask>);
    case 128: return many ? run(distill_kernel<T, 128, kMask, true>)
                          : run(distill_kernel<T, 128, kMask>);
    default: return run(distill_kernel<T, 256, kMask>);
  }
}

template <typename T>
int run_distill(const Rows& a, const DistillArgs& o, long long n, cudaStream_t st) {
  return a.mask ? run_distill_m<T, true>(a, o, n, st) : run_distill_m<T, false>(a, o, n, st);
}

}  // namespace lk
}  // namespace chm
