// Autograd of the losses in losses.cu.  A micro-batch's kernels take 12 us, so a step's time is the host's: 115 us through a Function in Python, 80 to 90 here, 50 of which torch's
// engine takes for any gradient.
#include <torch/extension.h>

namespace tk {

using OptT = c10::optional<torch::Tensor>;

std::vector<torch::Tensor> policy_loss_fwd(const torch::Tensor&, const torch::Tensor&, const torch::Tensor&, const OptT&, const OptT&, const OptT&, int64_t, int64_t, int64_t, double, double,
                                           double, double, double, double, double, int64_t, bool);
std::vector<torch::Tensor> policy_loss_bwd(const torch::Tensor&, const OptT&, const torch::Tensor&, const torch::Tensor&, double, int64_t, bool);
std::vector<torch::Tensor> preference_loss_fwd(const torch::Tensor&, const torch::Tensor&, const OptT&, int64_t, double, double, double, double, int64_t);
torch::Tensor preference_loss_bwd(const torch::Tensor&, const torch::Tensor&, const torch::Tensor&, int64_t);

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

static void no_second_derivative() { TORCH_CHECK(!at::GradMode::is_enabled(), "the loss kernels have no second derivative"); }
static torch::Tensor scalar_grad(const torch::Tensor& g) { return g.scalar_type() == torch::kFloat32 ? g : g.to(torch::kFloat32); }

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logps, const OptT& ent, const torch::Tensor& labels, const torch::Tensor& adv, const OptT& old, const OptT& ref,
                               int64_t ratio, int64_t kind, int64_t reduce, double eps_low, double eps_high, double beta, double entropy, double tau_pos, double tau_neg, double denominator,
                               int64_t ignore) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto out = policy_loss_fwd(logps, labels, adv, old, ref, ent, ratio, kind, reduce, eps_low, eps_high, beta, entropy, tau_pos, tau_neg, denominator, ignore, logps.requires_grad());
    ctx->save_for_backward({out[2], out[3], labels});
    ctx->saved_data["entropy"] = entropy;
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    no_second_derivative();
    const auto saved = ctx->get_saved_variables();
    const bool by_logps = ctx->needs_input_grad(0), by_ent = ctx->needs_input_grad(1);
    auto out = policy_loss_bwd(scalar_grad(g[0]), by_logps ? OptT(saved[0]) : OptT(), saved[1], saved[2], ctx->saved_data["entropy"].toDouble(), ctx->saved_data["ignore"].toInt(), by_ent);
    variable_list grads(17);
    if (by_logps) grads[0] = out[0];
    if (by_ent) grads[1] = out[1];
    return grads;
  }
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logps, const torch::Tensor& labels, const OptT& ref, int64_t form, double beta, double gamma, double smoothing,
                               double nll, int64_t ignore) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto out = preference_loss_fwd(logps, labels, ref, form, beta, gamma, smoothing, nll, ignore);
    ctx->save_for_backward({out[2], labels});
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    no_second_derivative();
    const auto saved = ctx->get_saved_variables();
    variable_list grads(9);
    grads[0] = preference_loss_bwd(scalar_grad(g[0]), saved[0], saved[1], ctx->saved_data["ignore"].toInt());
    return grads;
  }
};

std::vector<torch::Tensor> policy_loss(const torch::Tensor& logps, const OptT& ent, const torch::Tensor& labels, const torch::Tensor& adv, const OptT& old, const OptT& ref, int64_t ratio,
                                       int64_t kind, int64_t reduce, double eps_low, double eps_high, double beta, double entropy, double tau_pos, double tau_neg, double denominator,
                                       int64_t ignore) {
  return PolicyLoss::apply(logps, ent, labels, adv, old, ref, ratio, kind, reduce, eps_low, eps_high, beta, entropy, tau_pos, tau_neg, denominator, ignore);
}
std::vector<torch::Tensor> preference_loss(const torch::Tensor& logps, const torch::Tensor& labels, const OptT& ref, int64_t form, double beta, double gamma, double smoothing, double nll,
                                           int64_t ignore) {
  return PreferenceLoss::apply(logps, labels, ref, form, beta, gamma, smoothing, nll, ignore);
}

}  // namespace tk
