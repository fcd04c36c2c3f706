// chm_likelihood_f32.cu -- the likelihood and distillation kernels on fp32 logits.
#include "chm_likelihood_run.cuh"

namespace chm {
namespace lk {

template int run_log_probs<float>(const Rows&, const ScoreArgs&, long long, cudaStream_t);
template int run_log_probs_grad<float>(const Rows&, const ScoreGradArgs&, long long,
                                    cudaStream_t);
template int run_distill<float>(const Rows&, const DistillArgs&, long long, cudaStream_t);

int run_sum_rows(const float* row_loss, long long n, float* loss, cudaStream_t st) {
  ScopedLaunchTimer timer(kTimingScore, st);
  sum_rows_kernel<<<1, 1024, 0, st>>>(row_loss, n, loss);
  return launch_status();
}

}  // namespace lk
}  // namespace chm
