// chm_likelihood.cu -- C ABI of the likelihood and distillation operators
// (include/cherimoya_b200.h): argument checks and kernel dispatch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/cherimoya_b200.h"
#include "chm_host.h"
#include "chm_likelihood.h"

using namespace chm;

namespace {

#define LK_TRY(expr)               \
  do {                             \
    const int _s = (expr);         \
    if (_s != CHM_OK) return _s;   \
  } while (0)

size_t dtype_bytes(int dtype) { return dtype == CHM_LOGITS_F32 ? 4 : 2; }

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

int check_rows(const chm_rows* r, bool need_grad) {
  if (!r || r->n_examples < 0 || r->n_groups < 1 || !r->group_offset || !r->group_size)
    return CHM_ERR_INVALID_ARGUMENT;
  if (r->dtype < CHM_LOGITS_F32 || r->dtype > CHM_LOGITS_F16) return CHM_ERR_INVALID_ARGUMENT;
  if (!(r->temperature >= 1.f / 1024.f && r->temperature <= 1024.f))
    return CHM_ERR_INVALID_ARGUMENT;
  if (r->mask && !r->mask_group_offset) return CHM_ERR_INVALID_ARGUMENT;
  if (need_grad && !r->grad) return CHM_ERR_INVALID_ARGUMENT;
  if (r->grad && !r->grad_group_offset) return CHM_ERR_INVALID_ARGUMENT;
  bool empty = r->n_examples == 0;
  int largest = 0;
  for (int g = 0; g < r->n_groups; ++g) {
    if (r->group_size[g] < 0 || r->group_size[g] > CHM_ROW_MAX_ENTRIES)
      return CHM_ERR_INVALID_ARGUMENT;
    largest = std::max(largest, r->group_size[g]);
  }
  if (!empty && largest > 0) {
    if (!r->logits || misaligned(r->logits, dtype_bytes(r->dtype))) return CHM_ERR_INVALID_ARGUMENT;
    if (r->grad && misaligned(r->grad, dtype_bytes(r->dtype))) return CHM_ERR_INVALID_ARGUMENT;
  }
  // one block per row and launch: the grid's x extent
  if (r->n_examples > INT_MAX / std::min(r->n_groups, lk::kMaxGroups))
    return CHM_ERR_UNSUPPORTED;
  return CHM_OK;
}

// The launch's rows: groups [g0, g0 + ng).
lk::Rows make_rows(const chm_rows* r, int g0, int ng) {
  lk::Rows a{};
  a.z = r->logits;
  a.mask = r->mask;
  a.grad = r->grad;
  a.row_stride = r->row_stride;
  a.mask_stride = r->mask_row_stride;
  a.grad_stride = r->grad_row_stride;
  a.n_groups = r->n_groups;
  a.g0 = g0;
  a.ng = ng;
  a.t = r->temperature;
  a.inv_t = (float)(1.0 / (double)r->temperature);
  a.c = (float)(1.4426950408889634 / (double)r->temperature);   // log2(e) / T
  for (int g = 0; g < ng; ++g) {
    a.off[g] = r->group_offset[g0 + g];
    a.size[g] = r->group_size[g0 + g];
    if (r->mask) a.moff[g] = r->mask_group_offset[g0 + g];
    if (r->grad) a.goff[g] = r->grad_group_offset[g0 + g];
  }
  return a;
}

// Runs launch(rows, their number) for every run of up to kMaxGroups groups.
template <typename F>
int each_launch(const chm_rows* r, F launch) {
  launches_reset();
  if (r->n_examples == 0) return CHM_OK;
  for (int g0 = 0; g0 < r->n_groups; g0 += lk::kMaxGroups) {
    const lk::Rows a = make_rows(r, g0, std::min(lk::kMaxGroups, r->n_groups - g0));
    LK_TRY(launch(a, r->n_examples * a.ng));
  }
  return CHM_OK;
}

}  // namespace

extern "C" {

int32_t chm_log_probs(const chm_rows* rows, const int64_t* targets, int32_t n_targets,
                      int32_t top_k, float* log_probs, float* entropy, float* log_normalizer,
                      float* top_log_probs, int64_t* top_indices, float* stats,
                      chm_stream_t stream) {
  LK_TRY(check_rows(rows, false));
  if (n_targets < 0 || n_targets > CHM_ROW_MAX_TARGETS || top_k < 0 || top_k > CHM_ROW_MAX_TOP)
    return CHM_ERR_INVALID_ARGUMENT;
  if (rows->n_examples > 0 && ((n_targets > 0 && (!targets || !log_probs)) ||
                               (top_k > 0 && (!top_log_probs || !top_indices))))
    return CHM_ERR_INVALID_ARGUMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const lk::ScoreArgs o{reinterpret_cast<const long long*>(targets), n_targets, top_k, log_probs,
                        entropy, log_normalizer, top_log_probs,
                        reinterpret_cast<long long*>(top_indices), stats};
  return each_launch(rows, [&](const lk::Rows& a, long long n) {
    switch (rows->dtype) {
      case CHM_LOGITS_F32: return lk::run_log_probs<float>(a, o, n, st);
      case CHM_LOGITS_BF16: return lk::run_log_probs<__nv_bfloat16>(a, o, n, st);
      default: return lk::run_log_probs<__half>(a, o, n, st);
    }
  });
}

int32_t chm_log_probs_backward(const chm_rows* rows, const int64_t* targets, int32_t n_targets,
                               const int64_t* top_indices, int32_t top_k,
                               const float* stats, const float* entropy,
                               const float* g_log_probs, const float* g_entropy,
                               const float* g_log_normalizer, const float* g_top_log_probs,
                               chm_stream_t stream) {
  LK_TRY(check_rows(rows, true));
  if (n_targets < 0 || n_targets > CHM_ROW_MAX_TARGETS || top_k < 0 || top_k > CHM_ROW_MAX_TOP)
    return CHM_ERR_INVALID_ARGUMENT;
  if (rows->n_examples > 0 &&
      (!stats || (g_entropy && !entropy) || (n_targets > 0 && g_log_probs && !targets) ||
       (top_k > 0 && g_top_log_probs && !top_indices)))
    return CHM_ERR_INVALID_ARGUMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const lk::ScoreGradArgs o{reinterpret_cast<const long long*>(targets),
                            reinterpret_cast<const long long*>(top_indices), n_targets, top_k,
                            stats, entropy, n_targets > 0 ? g_log_probs : nullptr,
                            g_entropy, g_log_normalizer, top_k > 0 ? g_top_log_probs : nullptr};
  return each_launch(rows, [&](const lk::Rows& a, long long n) {
    switch (rows->dtype) {
      case CHM_LOGITS_F32: return lk::run_log_probs_grad<float>(a, o, n, st);
      case CHM_LOGITS_BF16: return lk::run_log_probs_grad<__nv_bfloat16>(a, o, n, st);
      default: return lk::run_log_probs_grad<__half>(a, o, n, st);
    }
  });
}

int32_t chm_distill(const chm_rows* rows, const int64_t* teacher_indices,
                    const float* teacher_log_probs, int32_t n_listed, int32_t renormalize,
                    const float* weight, float scale, const float* upstream,
                    int32_t upstream_stride, float* row_loss, float* loss, chm_stream_t stream) {
  LK_TRY(check_rows(rows, false));
  if (n_listed < 0 || n_listed > CHM_ROW_MAX_TARGETS || upstream_stride < 0 ||
      upstream_stride > 1 || (loss && !row_loss && rows->n_examples > 0))
    return CHM_ERR_INVALID_ARGUMENT;
  if (rows->n_examples > 0 && n_listed > 0 && (!teacher_indices || !teacher_log_probs))
    return CHM_ERR_INVALID_ARGUMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const lk::DistillArgs o{reinterpret_cast<const long long*>(teacher_indices), teacher_log_probs,
                          n_listed, renormalize != 0, weight, upstream, scale, upstream_stride,
                          row_loss};
  LK_TRY(each_launch(rows, [&](const lk::Rows& a, long long n) {
    switch (rows->dtype) {
      case CHM_LOGITS_F32: return lk::run_distill<float>(a, o, n, st);
      case CHM_LOGITS_BF16: return lk::run_distill<__nv_bfloat16>(a, o, n, st);
      default: return lk::run_distill<__half>(a, o, n, st);
    }
  }));
  if (loss) LK_TRY(lk::run_sum_rows(row_loss, rows->n_examples * rows->n_groups, loss, st));
  return CHM_OK;
}

}  // extern "C"
