// Autograd of the losses in losses.cu.  A micro-batch's kernels take 12 us, so a step's time is the host's: 115 us through a Function in Python, 85 to 110 here, 50 of which torch's
// engine takes for any gradient.
//
// The kernels have a first derivative only, for one gradient of the loss.  A call that asks for more (`twice`) keeps its inputs as they are, and a backward pass that is itself
// differentiated, or takes several gradients at once, runs the plain form of the operator on them (ops/reference.py).
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

// A call as it was made: its inputs with the versions that they had (the plain form would otherwise differentiate another call), the numbers of its rules, and its other numbers.  One entry:
// each costs a us.
static void keep(AutogradContext* ctx, const std::vector<OptT>& inputs, std::vector<int64_t> rules, std::vector<double> numbers) {
  std::vector<at::Tensor> tensors;
  std::vector<int64_t> versions;
  for (const auto& t : inputs) {
    tensors.push_back(t.has_value() ? *t : at::Tensor());
    versions.push_back(t.has_value() && t->defined() && !t->is_inference() ? t->_version() : 0);
  }
  ctx->saved_data["call"] = c10::ivalue::Tuple::create(std::move(tensors), std::move(versions), std::move(rules), std::move(numbers));
}
struct Call {
  std::vector<at::Tensor> inputs;
  std::vector<int64_t> rules;
  std::vector<double> numbers;
};
// Whether a backward pass wants what the kernels do not give
static bool plain_wanted(AutogradContext* ctx, const torch::Tensor& g) {
  const bool more = at::GradMode::is_enabled() || !g.has_storage();      // without storage: a wrapper of several
  TORCH_CHECK(!more || ctx->saved_data.count("call") != 0, "the loss kernels have no second derivative, and take one gradient of the loss");
  return more;
}
static Call kept(AutogradContext* ctx) {
  const auto call = ctx->saved_data["call"].toTuple();
  const auto& parts = call->elements();
  const auto versions = parts[1].toIntVector();
  Call c{parts[0].toTensorVector(), parts[2].toIntVector(), parts[3].toDoubleVector()};
  for (size_t i = 0; i < c.inputs.size(); ++i)
    TORCH_CHECK(!c.inputs[i].defined() || c.inputs[i].is_inference() || c.inputs[i]._version() == versions[i],
                "an input of a loss was modified by an inplace operation before its gradient was differentiated");
  return c;
}
// Gradients by the plain form: `form` of ops/reference.py with its arguments and the tensors that want one.  Errors come as C++ exceptions: the engine keeps them in threads without Python.
template <typename... A>
static variable_list plain_gradient(const char* form, const torch::Tensor& up, const std::vector<at::Tensor>& wanted, const A&... args) {
  namespace py = pybind11;
  py::gil_scoped_acquire gil;
  try {
    const auto out = py::module_::import("twinkle_b200.ops.reference").attr(form)(up, wanted, args...);
    return out.template cast<std::vector<at::Tensor>>();
  } catch (py::error_already_set& e) {
    const std::string what = e.what();
    e.restore();
    PyErr_Clear();
    TORCH_CHECK(false, what);
  }
}
static OptT given(const at::Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
static torch::Tensor scalar_grad(const torch::Tensor& g) { return g.scalar_type() == torch::kFloat32 ? g : g.to(torch::kFloat32); }

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logps, const OptT& ent, const torch::Tensor& labels, const torch::Tensor& adv, const OptT& old, const OptT& ref,
                               int64_t ratio, int64_t kind, int64_t reduce, double eps_low, double eps_high, double beta, double entropy, double tau_pos, double tau_neg, double denominator,
                               int64_t ignore, bool twice) {
    if (twice) keep(ctx, {logps, ent, labels, adv, old, ref}, {ratio, kind, reduce}, {eps_low, eps_high, beta, entropy, tau_pos, tau_neg, denominator});
    at::AutoDispatchBelowADInplaceOrView below;
    auto out = policy_loss_fwd(logps, labels, adv, old, ref, ent, ratio, kind, reduce, eps_low, eps_high, beta, entropy, tau_pos, tau_neg, denominator, ignore, logps.requires_grad());
    ctx->save_for_backward({out[2], out[3], labels});
    ctx->saved_data["entropy"] = entropy;
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const bool by_logps = ctx->needs_input_grad(0), by_ent = ctx->needs_input_grad(1);
    const int64_t ignore = ctx->saved_data["ignore"].toInt();
    variable_list grads(18);
    if (plain_wanted(ctx, g[0])) {
      const auto call = kept(ctx);
      const auto& x = call.inputs;       // log-probs, entropies, labels, advantages, old, reference
      std::vector<at::Tensor> wanted;
      if (by_logps) wanted.push_back(x[0]);
      if (by_ent) wanted.push_back(x[1]);
      const auto out = plain_gradient("policy_loss_gradient", g[0], wanted, x[0], x[2], x[3], given(x[4]), given(x[5]), given(x[1]), call.rules, call.numbers, ignore);
      if (by_logps) grads[0] = out[0];
      if (by_ent) grads[1] = out[by_logps ? 1 : 0];
      return grads;
    }
    const auto saved = ctx->get_saved_variables();
    auto out = policy_loss_bwd(scalar_grad(g[0]), by_logps ? OptT(saved[0]) : OptT(), saved[1], saved[2], ctx->saved_data["entropy"].toDouble(), ignore, by_ent);
    if (by_logps) grads[0] = out[0];
    if (by_ent) grads[1] = out[1];
    return grads;
  }
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logps, const torch::Tensor& labels, const OptT& ref, int64_t form, double beta, double gamma, double smoothing,
                               double nll, int64_t ignore, bool twice) {
    if (twice) keep(ctx, {logps, labels, ref}, {form}, {beta, gamma, smoothing, nll});
    at::AutoDispatchBelowADInplaceOrView below;
    auto out = preference_loss_fwd(logps, labels, ref, form, beta, gamma, smoothing, nll, ignore);
    ctx->save_for_backward({out[2], labels});
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list grads(10);
    if (plain_wanted(ctx, g[0])) {
      const auto call = kept(ctx);
      const auto& x = call.inputs;
      grads[0] = plain_gradient("preference_loss_gradient", g[0], {x[0]}, x[0], x[1], given(x[2]), call.rules[0], call.numbers, ctx->saved_data["ignore"].toInt())[0];
      return grads;
    }
    const auto saved = ctx->get_saved_variables();
    grads[0] = preference_loss_bwd(scalar_grad(g[0]), saved[0], saved[1], ctx->saved_data["ignore"].toInt());
    return grads;
  }
};

std::vector<torch::Tensor> policy_loss(const torch::Tensor& logps, const OptT& ent, const torch::Tensor& labels, const torch::Tensor& adv, const OptT& old, const OptT& ref, int64_t ratio,
                                       int64_t kind, int64_t reduce, double eps_low, double eps_high, double beta, double entropy, double tau_pos, double tau_neg, double denominator,
                                       int64_t ignore, bool twice) {
  return PolicyLoss::apply(logps, ent, labels, adv, old, ref, ratio, kind, reduce, eps_low, eps_high, beta, entropy, tau_pos, tau_neg, denominator, ignore, twice);
}
std::vector<torch::Tensor> preference_loss(const torch::Tensor& logps, const torch::Tensor& labels, const OptT& ref, int64_t form, double beta, double gamma, double smoothing, double nll,
                                           int64_t ignore, bool twice) {
  return PreferenceLoss::apply(logps, labels, ref, form, beta, gamma, smoothing, nll, ignore, twice);
}

}  // namespace tk
