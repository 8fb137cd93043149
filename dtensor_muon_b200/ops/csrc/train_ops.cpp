// Registrations of the decoder's training operators for CUDA tensors: the kernels, and their
// gradients as autograd functions in C++ (a Python formula would cost more host time than the
// small calls take). The schemas, the CPU and the fake kernels are in ops/library.py. Each
// autograd function calls its operators through the dispatcher, so that tracers see them.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <atomic>

#include "train_ops.h"

namespace dmb {

namespace {
std::atomic<int64_t> g_launches{0};
}

void count_launches(int64_t n) { g_launches.fetch_add(n, std::memory_order_relaxed); }
int64_t launches_counted() { return g_launches.load(std::memory_order_relaxed); }

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor saved(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": no gradient of the gradient (create_graph=True)");
}

#define DMB_OP(var, name, type) \
  static const auto var = c10::Dispatcher::singleton().findSchemaOrThrow("dmb::" name, "").typed<type>()

// ------------------------------------------------------------- qk_norm_rope
using QkFwd = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                         const Tensor&, const OptTensor&, double);
using QkBwd = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                         const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                         const OptTensor&, double, bool);

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                               const Tensor& cos, const Tensor& sin, const OptTensor& positions, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    DMB_OP(op, "qk_norm_rope", QkFwd);
    auto [qo, ko] = op.call(q, k, qw, kw, cos, sin, positions, eps);
    ctx->save_for_backward({q, k, qw, kw, cos, sin, saved(positions)});
    ctx->saved_data["eps"] = eps;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("qk_norm_rope");
    const auto s = ctx->get_saved_variables();
    const bool weights = ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    DMB_OP(op, "qk_norm_rope_backward", QkBwd);
    auto [dq, dk, dqw, dkw] = op.call(g[0], g[1], s[0], s[1], s[2], s[3], s[4], s[5], maybe(s[6]),
                                      ctx->saved_data["eps"].toDouble(), weights);
    return {dq, dk, weights ? dqw : Tensor(), weights ? dkw : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope_autograd(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                                                 const Tensor& cos, const Tensor& sin, const OptTensor& positions, double eps) {
  auto r = QkNormRope::apply(q, k, qw, kw, cos, sin, positions, eps);
  return {r[0], r[1]};
}

// -------------------------------------------------------------------- route
using RouteFwd = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(const Tensor&, int64_t, const OptTensor&);
using RouteBwd = Tensor(const OptTensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&, const Tensor&,
                        const OptTensor&);

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t top_k, const OptTensor& mask) {
    at::AutoDispatchBelowADInplaceOrView below;
    DMB_OP(op, "route", RouteFwd);
    auto [gates, experts, counts, balance, z] = op.call(logits, top_k, mask);
    ctx->mark_non_differentiable({experts, counts});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, experts, counts, saved(mask)});
    return {gates, experts, counts, balance, z};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("route");
    const auto s = ctx->get_saved_variables();
    DMB_OP(op, "route_backward", RouteBwd);
    return {op.call(maybe(g[0]), maybe(g[3]), maybe(g[4]), s[0], s[1], s[2], maybe(s[3])), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_autograd(const Tensor& logits, int64_t top_k, const OptTensor& mask) {
  auto r = Route::apply(logits, top_k, mask);
  return {r[0], r[1], r[2], r[3], r[4]};
}

// ----------------------------------------- token_logprobs and its two losses
using LogprobFwd = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&);
using PolicyFwd = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&,
                                                                            const Tensor&, const OptTensor&,
                                                                            const OptTensor&, double, double, double);
using PreferenceFwd = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&,
                                                                        const OptTensor&, double, double);
using LogprobBwd = Tensor(const Tensor&, const OptTensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&);

Tensor logprob_grad(const Tensor& coef, const OptTensor& scale, const Tensor& logits, const Tensor& targets,
                    const Tensor& stats, const OptTensor& mask) {
  DMB_OP(op, "token_logprobs_backward", LogprobBwd);
  return op.call(coef, scale, logits, targets, stats, mask);
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, const OptTensor& mask) {
    at::AutoDispatchBelowADInplaceOrView below;
    DMB_OP(op, "token_logprobs", LogprobFwd);
    auto [logp, stats] = op.call(logits, targets, mask);
    ctx->mark_non_differentiable({stats});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, stats, saved(mask)});
    return {logp, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("token_logprobs");
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    return {logprob_grad(g[0], {}, s[0], s[1], s[2], maybe(s[3])), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> token_logprobs_autograd(const Tensor& logits, const Tensor& targets, const OptTensor& mask) {
  auto r = TokenLogprobs::apply(logits, targets, mask);
  return {r[0], r[1]};
}

// A token's gradient needs nothing but that token's logp, so that the forward kernel can write the logits' gradient while
// it has the row at hand, and the logits are read once instead of twice. It does so for a loss gradient of 1, which is
// what backward() starts with; the backward pass then only looks at that value, and computes all of it where it is another.
// The gradient is handed out once: a second backward pass of a retained graph computes its own. Not where a tracer or a
// graph capture looks on, which would take the two passes apart.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, const Tensor& old_logp,
                               const Tensor& advantages, const OptTensor& ref_logp, const OptTensor& mask, double clip_low,
                               double clip_high, double kl_coef, bool grad_now) {
    at::AutoDispatchBelowADInplaceOrView below;
    DMB_OP(op, "policy_loss", PolicyFwd);
    Tensor grad;
    auto [loss, logp, kl, clipped, stats, coef] =
        grad_now ? policy_loss_fwd_grad(logits, targets, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef, &grad)
                 : op.call(logits, targets, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef);
    if (grad.defined()) ctx->saved_data["grad"] = grad;
    ctx->mark_non_differentiable({logp, kl, clipped, stats, coef});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, stats, coef, saved(mask)});
    return {loss, logp, kl, clipped, stats, coef};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("policy_loss");
    variable_list out(10);
    if (!g[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto ready = ctx->saved_data.find("grad");
    if (ready == ctx->saved_data.end()) {
      out[0] = logprob_grad(s[3], g[0], s[0], s[1], s[2], maybe(s[4]));
    } else {
      out[0] = token_logprobs_bwd_ready(s[3], g[0], s[0], s[1], s[2], maybe(s[4]), ready->second.toTensor());
      ctx->saved_data.erase(ready);
    }
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> policy_loss_autograd(
    const Tensor& logits, const Tensor& targets, const Tensor& old_logp, const Tensor& advantages, const OptTensor& ref_logp,
    const OptTensor& mask, double clip_low, double clip_high, double kl_coef) {
  const auto keys = logits.key_set();
  const bool plain = !keys.has(c10::DispatchKey::Python) && !keys.has(c10::DispatchKey::Functionalize) &&
                     !c10::impl::TorchDispatchModeTLS::any_modes_set();
  bool grad_now = plain && at::GradMode::is_enabled() && logits.requires_grad();
  if (grad_now) {
    const c10::cuda::CUDAGuard guard(logits.device());
    grad_now = c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None;
  }
  auto r = PolicyLoss::apply(logits, targets, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef, grad_now);
  return {r[0], r[1], r[2], r[3], r[4], r[5]};
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, const Tensor& ref_logp,
                               const OptTensor& mask, double beta, double label_smoothing) {
    at::AutoDispatchBelowADInplaceOrView below;
    DMB_OP(op, "preference_loss", PreferenceFwd);
    auto [loss, logp, rewards, stats, coef] = op.call(logits, targets, ref_logp, mask, beta, label_smoothing);
    ctx->mark_non_differentiable({logp, rewards, stats, coef});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, stats, coef, saved(mask)});
    return {loss, logp, rewards, stats, coef};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("preference_loss");
    variable_list out(6);
    if (!g[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = logprob_grad(s[3], g[0], s[0], s[1], s[2], maybe(s[4]));
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> preference_loss_autograd(const Tensor& logits, const Tensor& targets,
                                                                            const Tensor& ref_logp, const OptTensor& mask,
                                                                            double beta, double label_smoothing) {
  auto r = PreferenceLoss::apply(logits, targets, ref_logp, mask, beta, label_smoothing);
  return {r[0], r[1], r[2], r[3], r[4]};
}

}  // namespace

TORCH_LIBRARY_IMPL(dmb, CUDA, m) {
  m.impl("qk_norm_rope", qk_norm_rope_fwd);
  m.impl("qk_norm_rope_backward", qk_norm_rope_bwd);
  m.impl("route", route_fwd);
  m.impl("route_backward", route_bwd);
  m.impl("token_logprobs", token_logprobs_fwd);
  m.impl("token_logprobs_backward", token_logprobs_bwd);
  m.impl("policy_loss", policy_loss_fwd);
  m.impl("preference_loss", preference_loss_fwd);
}

TORCH_LIBRARY_IMPL(dmb, AutogradCUDA, m) {
  m.impl("qk_norm_rope", qk_norm_rope_autograd);
  m.impl("route", route_autograd);
  m.impl("token_logprobs", token_logprobs_autograd);
  m.impl("policy_loss", policy_loss_autograd);
  m.impl("preference_loss", preference_loss_autograd);
}

}  // namespace dmb
