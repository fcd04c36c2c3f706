// chm_likelihood_f16.cu -- the likelihood and distillation kernels on fp16 logits.
#include "chm_likelihood_run.cuh"

namespace chm {
namespace lk {

template int run_log_probs<__half>(const Rows&, const ScoreArgs&, long long, cudaStream_t);
template int run_log_probs_grad<__half>(const Rows&, const ScoreGradArgs&, long long,
                                    cudaStream_t);
template int run_distill<__half>(const Rows&, const DistillArgs&, long long, cudaStream_t);

}  // namespace lk
}  // namespace chm
