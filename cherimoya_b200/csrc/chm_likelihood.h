// chm_likelihood.h -- kernel parameters and launch functions of the likelihood
// and distillation operators. Each logits type has its own translation unit.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace chm {
namespace lk {

constexpr int kMaxGroups = 64;      // groups of one launch (kernel parameters)
constexpr int kMaxList = 1024;      // given / listed entries per row
constexpr int kMaxTop = 128;

struct Rows {
  const void* z;
  const uint8_t* mask;
  void* grad;
  long long row_stride, mask_stride, grad_stride;
  int n_groups, g0, ng;             // groups in all; this launch's first and count
  float c;                          // log2(e) / T
  float inv_t, t;
  long long off[kMaxGroups], moff[kMaxGroups], goff[kMaxGroups];
  int size[kMaxGroups];
};

struct ScoreArgs {
  const long long* targets;
  int n_targets, top_k;
  float *log_probs, *entropy, *log_norm, *top_log_probs;
  long long* top_indices;
  float* stats;
};

struct ScoreGradArgs {
  const long long *targets, *top_indices;
  int n_targets, top_k;
  const float *stats, *entropy, *g_log_probs, *g_entropy, *g_log_norm, *g_top;
};

struct DistillArgs {
  const long long* indices;
  const float* log_probs;
  int n_listed, renormalize;
  const float *weight, *upstream;
  float scale;
  int upstream_stride;
  float* row_loss;
};

// Each launches over the n rows of one launch and returns a chm_status.
template <typename T>
int run_log_probs(const Rows& a, const ScoreArgs& o, long long n, cudaStream_t st);
template <typename T>
int run_log_probs_grad(const Rows& a, const ScoreGradArgs& o, long long n, cudaStream_t st);
template <typename T>
int run_distill(const Rows& a, const DistillArgs& o, long long n, cudaStream_t st);
int run_sum_rows(const float* row_loss, long long n, float* loss, cudaStream_t st);

}  // namespace lk
}  // namespace chm
