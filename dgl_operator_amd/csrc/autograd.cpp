// Autograd of the typed-row operators and of log_probs on the GPU, in C++: a
// pass over few rows is bound by the host, and a backward pass that stays out
// of Python costs a fraction of one that does not.

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace doa {

at::Tensor dispatch_rows(at::Tensor x, at::Tensor position,
                         at::Tensor offsets);
at::Tensor combine_rows(at::Tensor y, at::Tensor position,
                        c10::optional<at::Tensor> weights);
std::tuple<at::Tensor, at::Tensor> combine_rows_bwd(
    at::Tensor gout, c10::optional<at::Tensor> y, at::Tensor position,
    at::Tensor offsets, c10::optional<at::Tensor> weights, bool want_y);
at::Tensor segment_mm(at::Tensor offsets, at::Tensor x, at::Tensor weight,
                      bool transposed);
at::Tensor segment_mm_wgrad(at::Tensor offsets, at::Tensor x, at::Tensor grad);
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
log_probs_fwd(at::Tensor logits, c10::optional<at::Tensor> target, int64_t k,
              int64_t ignore);
at::Tensor log_probs_bwd(at::Tensor logits, c10::optional<at::Tensor> target,
                         int64_t ignore, at::Tensor top_idx, at::Tensor stats,
                         at::Tensor ent, c10::optional<at::Tensor> g_lp,
                         c10::optional<at::Tensor> g_ent,
                         c10::optional<at::Tensor> g_top);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::Variable;
using torch::autograd::variable_list;

using Maybe = c10::optional<at::Tensor>;

Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

// gradients that refuse to be differentiated once more
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list held, out(grads.size());
  for (auto& g : grads)
    if (g.defined()) held.push_back(g.detach().requires_grad_(true));
  if (held.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that has one derivative only",
      held.size());
  held = (*error)(std::move(held));
  size_t next = 0;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) out[i] = held[next++];
  return out;
}

struct DispatchRows : Function<DispatchRows> {
  static Variable forward(AutogradContext* ctx, const Variable& x,
                          const Variable& position, const Variable& offsets) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({position});
    return dispatch_rows(x, position, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return {Variable(), Variable(), Variable()};
    variable_list out;
    {
      at::AutoGradMode off(false);
      out = {combine_rows(g[0], ctx->get_saved_variables()[0], c10::nullopt),
             Variable(), Variable()};
    }
    return once(std::move(out));
  }
};

struct CombineRows : Function<CombineRows> {
  static Variable forward(AutogradContext* ctx, const Variable& y,
                          const Maybe& weights, const Variable& position,
                          const Variable& offsets) {
    ctx->set_materialize_grads(false);
    // the weights act in 32 bits whatever they come in
    at::Tensor w;
    if (weights.has_value()) w = weights->to(at::kFloat).contiguous();
    const bool want_w = weights.has_value() && weights->requires_grad();
    if (weights.has_value())
      ctx->saved_data["type"] = (int64_t)weights->scalar_type();
    ctx->save_for_backward({want_w ? y : Variable(), w, position, offsets});
    return combine_rows(y, position, maybe(w));
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined())
      return {Variable(), Variable(), Variable(), Variable()};
    variable_list out(4);
    {
      at::AutoGradMode off(false);
      const auto s = ctx->get_saved_variables();
      // y has the graph's first edge, the weights, if there are any, its second
      const bool want_y = ctx->needs_input_grad(0);
      const bool want_w = s[0].defined() && ctx->needs_input_grad(1);
      auto [dy, dw] = combine_rows_bwd(g[0], want_w ? Maybe(s[0]) : Maybe(),
                                       s[2], s[3], maybe(s[1]), want_y);
      out[0] = dy;
      if (dw.defined())
        out[1] = dw.to((at::ScalarType)ctx->saved_data["type"].toInt());
    }
    return once(std::move(out));
  }
};

struct SegmentMM : Function<SegmentMM> {
  static Variable forward(AutogradContext* ctx, const Variable& offsets,
                          const Variable& x, const Variable& weight) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({offsets, weight.requires_grad() ? x : Variable(),
                            x.requires_grad() ? weight : Variable()});
    return segment_mm(offsets, x, weight, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(3);
    if (!g[0].defined()) return out;
    {
      at::AutoGradMode off(false);
      const auto s = ctx->get_saved_variables();
      // (the graph's edges: offsets, x, weight)
      if (s[2].defined() && ctx->needs_input_grad(1))
        out[1] = segment_mm(s[0], g[0], s[2], true);
      if (s[1].defined() && ctx->needs_input_grad(2))
        out[2] = segment_mm_wgrad(s[0], s[1], g[0]);
    }
    return once(std::move(out));
  }
};

// outputs: entropy, top_log_prob, top_index and, with a target, log_prob
struct LogProbs : Function<LogProbs> {
  static variable_list forward(AutogradContext* ctx, const Variable& logits,
                               const Maybe& target, int64_t k, int64_t ignore) {
    ctx->set_materialize_grads(false);
    auto [lp, ent, top, index, stats] = log_probs_fwd(logits, target, k, ignore);
    ctx->saved_data["ignore"] = ignore;
    ctx->save_for_backward({logits, target.has_value() ? *target : Variable(),
                            index, stats, ent});
    ctx->mark_non_differentiable({index});
    variable_list out = {ent, top, index};
    if (lp.defined()) out.push_back(lp);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(4);
    {
      at::AutoGradMode off(false);
      const auto s = ctx->get_saved_variables();
      out[0] = log_probs_bwd(
          s[0], maybe(s[1]), ctx->saved_data["ignore"].toInt(), s[2], s[3],
          s[4], g.size() > 3 ? maybe(g[3]) : Maybe(), maybe(g[0]), maybe(g[1]));
    }
    return once(std::move(out));
  }
};

}  // namespace

at::Tensor dispatch_rows_ad(at::Tensor x, at::Tensor position,
                            at::Tensor offsets) {
  return DispatchRows::apply(x, position, offsets);
}

at::Tensor combine_rows_ad(at::Tensor y, Maybe weights, at::Tensor position,
                           at::Tensor offsets) {
  return CombineRows::apply(y, weights, position, offsets);
}

at::Tensor segment_mm_ad(at::Tensor offsets, at::Tensor x, at::Tensor weight) {
  return SegmentMM::apply(offsets, x, weight);
}

std::vector<at::Tensor> log_probs_ad(at::Tensor logits, Maybe target, int64_t k,
                                     int64_t ignore) {
  return LogProbs::apply(logits, target, k, ignore);
}

}  // namespace doa
