// Host entry points of the decoder's training operators (qk_norm_rope.cu,
// route.cu, logprob_loss.cu), called by their registrations in train_ops.cpp.
#pragma once

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/util/Optional.h>

#include <tuple>

namespace dmb {

using OptTensor = c10::optional<at::Tensor>;

// A contiguous tensor on `like`'s device, without the way through the dispatcher: of a small call's host time each
// allocation is a good part.
inline at::Tensor new_empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

int* device_error_word(int dev);
void count_launches(int64_t n);  // kernels launched by these operators, for ops/_ext.py's counter
int64_t launches_counted();

// ---- qk_norm_rope.cu
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                                                    const at::Tensor& k_weight, const at::Tensor& cos,
                                                    const at::Tensor& sin, const OptTensor& positions, double eps);
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_bwd(
    const at::Tensor& dq_out, const at::Tensor& dk_out, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& q_weight, const at::Tensor& k_weight, const at::Tensor& cos, const at::Tensor& sin,
    const OptTensor& positions, double eps, bool weight_grads);

// ---- route.cu
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> route_fwd(const at::Tensor& logits,
                                                                                int64_t top_k, const OptTensor& mask);
at::Tensor route_bwd(const OptTensor& dgates, const OptTensor& dbalance, const OptTensor& dz, const at::Tensor& logits,
                     const at::Tensor& experts, const at::Tensor& counts, const OptTensor& mask);

// ---- logprob_loss.cu
std::tuple<at::Tensor, at::Tensor> token_logprobs_fwd(const at::Tensor& logits, const at::Tensor& targets,
                                                      const OptTensor& mask);
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> policy_loss_fwd(
    const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& old_logp, const at::Tensor& advantages,
    const OptTensor& ref_logp, const OptTensor& mask, double clip_low, double clip_high, double kl_coef);
// As policy_loss_fwd; where the kernels can, they also put the logits' gradient for a loss gradient of 1 into *grad.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> policy_loss_fwd_grad(
    const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& old_logp, const at::Tensor& advantages,
    const OptTensor& ref_logp, const OptTensor& mask, double clip_low, double clip_high, double kl_coef, at::Tensor* grad);
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> preference_loss_fwd(
    const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& ref_logp, const OptTensor& mask, double beta,
    double label_smoothing);
at::Tensor token_logprobs_bwd(const at::Tensor& coef, const OptTensor& scale, const at::Tensor& logits,
                              const at::Tensor& targets, const at::Tensor& stats, const OptTensor& mask);
// As token_logprobs_bwd; `ready`, where defined, holds the gradient for a scale of 1, and is returned with that for `scale`.
at::Tensor token_logprobs_bwd_ready(const at::Tensor& coef, const OptTensor& scale, const at::Tensor& logits,
                                    const at::Tensor& targets, const at::Tensor& stats, const OptTensor& mask,
                                    const at::Tensor& ready);

}  // namespace dmb
