// chm_likelihood_bf16.cu -- the likelihood and distillation kernels on bf16 logits.
#include "chm_likelihood_run.cuh"

namespace chm {
namespace lk {

template int run_log_probs<__nv_bfloat16>(const Rows&, const ScoreArgs&, long long, cudaStream_t);
template int run_log_probs_grad<__nv_bfloat16>(const Rows&, const ScoreGradArgs&, long long,
                                    cudaStream_t);
template int run_distill<__nv_bfloat16>(const Rows&, const DistillArgs&, long long, cudaStream_t);

}  // namespace lk
}  // namespace chm
