// chm_likelihood_f32.cu -- the likelihood and distillation kernels on fp32 logits.
#include "chm_likelihood_run.cuh"

namespace chm {
namespace lk {

template int run_log_probs<float>(const Rows&, const ScoreArgs&, long long, cudaStream_t);
template int run_log_probs_grad<float>(const Rows&, const ScoreGradArgs&, long long,
                                    cudaStream_t);
template int run_distill<float>(const Rows&, const DistillArgs&, long long, cudaStream_t);

int run_sum_rows(const float* row_loss, long long n, float* loss, cudaStream_t st) {
  // may start while the rows' kernel ends; it waits for that kernel's writes itself
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ScopedLaunchTimer timer(kTimingScore, st);
  cudaLaunchKernelEx(&cfg, sum_rows_kernel, row_loss, n, loss);
  return launch_status();
}

}  // namespace lk
}  // namespace chm
