// Operators and autograd nodes of the attentional operators.
//
// The nodes are C++: a training call on a small batch costs its host time
// (a Python node's backward takes the interpreter lock in the engine's
// device thread: 91 us a forward + backward of match_log_probs on 64 x 19
// scores, of which the kernels are 9).
#include "attentional.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

namespace dgmc {

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor& t) { return t.has_value() && wants(*t); }

bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool dual(const OptTensor& t) { return t.has_value() && dual(*t); }

// (A tangent is refused: these nodes, and the calls that need none, know no
// forward mode and would drop it.)
template <typename... A>
bool wants_grad(const char* name, const A&... a) {
  TORCH_CHECK(!(dual(a) || ...), name,
              ": forward-mode differentiation is not supported");
  return at::GradMode::is_enabled() && (wants(a) || ...);
}

OptTensor opt(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}
Tensor def(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// Gradients that cannot be differentiated again (create_graph = True): the
// error comes where a second backward reaches them.
variable_list once(variable_list g) {
  if (!at::GradMode::is_enabled()) return g;
  variable_list in;
  for (auto& t : g) in.push_back(t.defined() ? t.detach() : t);
  for (auto& t : in)
    if (t.defined() && t.is_floating_point()) t.requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "this operator's gradient cannot be differentiated again",
      (int64_t)in.size());
  return (*error)(std::move(in));
}

// --------------------------------------------------------------------------
struct SegmentAttention
    : public torch::autograd::Function<SegmentAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q,
                        const Tensor& k, const Tensor& v,
                        const OptTensor& bias, const Tensor& ptr_q,
                        const Tensor& ptr_k, const OptTensor& pos_q,
                        const OptTensor& pos_k, double scale, double cap,
                        int64_t half, int64_t mbits, double dmax, bool x6) {
    auto [out, lo, stat] =
        segattn::forward(q, k, v, ptr_q, ptr_k, scale, cap, bias, pos_q,
                         pos_k, {half, mbits, dmax}, x6, true);
    ctx->save_for_backward({q, k, v, def(bias), ptr_q, ptr_k, def(pos_q),
                            def(pos_k), out, lo, stat});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    ctx->saved_data["half"] = half;
    ctx->saved_data["mbits"] = mbits;
    ctx->saved_data["dmax"] = dmax;
    ctx->saved_data["x6"] = x6;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    Tensor grad = g[0];
    if (grad.size(-1) != 1 && grad.stride(-1) != 1) grad = grad.contiguous();
    auto& d = ctx->saved_data;
    auto [dq, dk, dv, db] = segattn::backward(
        grad, s[0], s[1], s[2], s[8], s[9], s[10], s[4], s[5],
        d["scale"].toDouble(), d["cap"].toDouble(), opt(s[3]), opt(s[6]),
        opt(s[7]),
        {d["half"].toInt(), d["mbits"].toInt(), d["dmax"].toDouble()},
        d["x6"].toBool());
    variable_list r = once({dq, dk, dv, s[3].defined() ? db : Tensor()});
    r.resize(14);
    return r;
  }
};

Tensor segment_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                         const OptTensor& bias, const Tensor& ptr_q,
                         const Tensor& ptr_k, const OptTensor& pos_q,
                         const OptTensor& pos_k, double scale, double cap,
                         int64_t half, int64_t mbits, double dmax, bool x6) {
  return std::get<0>(segattn::forward(q, k, v, ptr_q, ptr_k, scale, cap, bias,
                                      pos_q, pos_k, {half, mbits, dmax},
                                      x6, false));
}

Tensor segment_attention_autograd(const Tensor& q, const Tensor& k,
                                  const Tensor& v, const OptTensor& bias,
                                  const Tensor& ptr_q, const Tensor& ptr_k,
                                  const OptTensor& pos_q,
                                  const OptTensor& pos_k, double scale,
                                  double cap, int64_t half, int64_t mbits,
                                  double dmax, bool x6) {
  if (wants_grad("segment_attention", q, k, v, bias))
    return SegmentAttention::apply(q, k, v, bias, ptr_q, ptr_k, pos_q, pos_k,
                                   scale, cap, half, mbits, dmax, x6);
  at::AutoDispatchBelowADInplaceOrView below;
  return segment_attention(q, k, v, bias, ptr_q, ptr_k, pos_q, pos_k, scale,
                           cap, half, mbits, dmax, x6);
}

// --------------------------------------------------------------------------
struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const OptTensor& residual,
                               const OptTensor& weight, const OptTensor& bias,
                               double eps) {
    auto [y, s, stat] = layer_norm_fwd(x, residual, weight, bias, eps, true);
    ctx->save_for_backward(
        {residual.has_value() ? s : x, def(weight), stat});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->set_materialize_grads(false);
    return residual.has_value() ? variable_list{y, s} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const Tensor ds = residual ? g[1] : Tensor();
    Tensor dx = ds, dw, db;
    if (g[0].defined()) {
      std::tie(dx, dw, db) = layer_norm_bwd(
          g[0], opt(ds), s[0], s[2], opt(s[1]), s[1].defined());
      if (!s[1].defined()) dw = Tensor();
      if (!ctx->saved_data["bias"].toBool()) db = Tensor();
    }
    variable_list r = once({dx, residual ? dx : Tensor(), dw, db});
    r.resize(5);
    return r;
  }
};

std::vector<Tensor> layer_norm(const Tensor& x, const OptTensor& residual,
                               const OptTensor& weight, const OptTensor& bias,
                               double eps) {
  auto [y, s, stat] = layer_norm_fwd(x, residual, weight, bias, eps, false);
  return residual.has_value() ? std::vector<Tensor>{y, s}
                              : std::vector<Tensor>{y};
}

std::vector<Tensor> layer_norm_autograd(const Tensor& x,
                                        const OptTensor& residual,
                                        const OptTensor& weight,
                                        const OptTensor& bias, double eps) {
  if (wants_grad("layer_norm", x, residual, weight, bias))
    return LayerNorm::apply(x, residual, weight, bias, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  return layer_norm(x, residual, weight, bias, eps);
}

// --------------------------------------------------------------------------
struct MatchLogProb : public torch::autograd::Function<MatchLogProb> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z,
                               const Tensor& y, const OptTensor& n,
                               int64_t k) {
    auto [logp, ent, top_lp, top_idx, stat] =
        match_logprob_fwd(z, y, n, k, true);
    ctx->save_for_backward({z, y, def(n), logp, ent, stat});
    ctx->mark_non_differentiable({top_lp, top_idx});
    ctx->set_materialize_grads(false);
    return {logp, ent, top_lp, top_idx};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined() && !g[1].defined()) return variable_list(4);
    OptTensor gl, gh;
    if (g[0].defined()) gl = g[0].to(at::kFloat).contiguous();
    if (g[1].defined()) gh = g[1].to(at::kFloat).contiguous();
    variable_list r = once({match_logprob_bwd(gl, gh, s[0], s[1], opt(s[2]),
                                              s[3], s[4], s[5])});
    r.resize(4);
    return r;
  }
};

std::vector<Tensor> match_logprob(const Tensor& z, const Tensor& y,
                                  const OptTensor& n, int64_t k) {
  auto [logp, ent, top_lp, top_idx, stat] =
      match_logprob_fwd(z, y, n, k, false);
  return {logp, ent, top_lp, top_idx};
}

std::vector<Tensor> match_logprob_autograd(const Tensor& z, const Tensor& y,
                                           const OptTensor& n, int64_t k) {
  if (wants_grad("match_log_probs", z)) return MatchLogProb::apply(z, y, n, k);
  at::AutoDispatchBelowADInplaceOrView below;
  return match_logprob(z, y, n, k);
}

}  // namespace

}  // namespace dgmc

TORCH_LIBRARY_FRAGMENT(dgmc_amd, m) {
  m.def(
      "segment_attention(Tensor q, Tensor k, Tensor v, Tensor? bias, Tensor "
      "ptr_q, Tensor ptr_k, Tensor? pos_q, Tensor? pos_k, float scale, float "
      "cap, int half, int mbits, float dmax, bool x6) -> Tensor");
  m.def(
      "layer_norm(Tensor x, Tensor? residual, Tensor? weight, Tensor? bias, "
      "float eps) -> Tensor[]");
  m.def(
      "match_logprob(Tensor z, Tensor y, Tensor? n, int k) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(dgmc_amd, CUDA, m) {
  m.impl("segment_attention", &dgmc::segment_attention);
  m.impl("layer_norm", &dgmc::layer_norm);
  m.impl("match_logprob", &dgmc::match_logprob);
}

TORCH_LIBRARY_IMPL(dgmc_amd, AutogradCUDA, m) {
  m.impl("segment_attention", &dgmc::segment_attention_autograd);
  m.impl("layer_norm", &dgmc::layer_norm_autograd);
  m.impl("match_logprob", &dgmc::match_logprob_autograd);
}
