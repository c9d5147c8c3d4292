// Autograd nodes of the sequence-model operators.  They are C++ so that a
// training step spends its host time on launches: a Python node costs more
// than the smaller of these kernels.

#include <torch/extension.h>
#include <c10/hip/HIPGraphsC10Utils.h>

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

torch::Tensor embed_lookup(torch::Tensor ids, torch::Tensor w, double scale,
                           bool has_ignore, long ignore);
torch::Tensor embed_grad(torch::Tensor ids, torch::Tensor gy, long vocab,
                         double scale, bool has_ignore, long ignore);
torch::Tensor dropout(torch::Tensor x, torch::Tensor key, long threshold,
                      double scale);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> rms_norm_fwd(
    torch::Tensor x, torch::Tensor w, c10::optional<torch::Tensor> res,
    double eps);
std::tuple<torch::Tensor, torch::Tensor> rms_norm_bwd(
    torch::Tensor gy, torch::Tensor x, c10::optional<torch::Tensor> res,
    c10::optional<torch::Tensor> gh, torch::Tensor w, torch::Tensor rstd);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> linear_attention_fwd(
    torch::Tensor q, torch::Tensor k, torch::Tensor v,
    torch::Tensor log_decay, c10::optional<torch::Tensor> first,
    c10::optional<torch::Tensor> lengths, double scale);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
linear_attention_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                     torch::Tensor log_decay,
                     c10::optional<torch::Tensor> first,
                     c10::optional<torch::Tensor> lengths, double scale,
                     torch::Tensor states, torch::Tensor go,
                     c10::optional<torch::Tensor> glast, bool need_q,
                     bool need_k, bool need_v, bool need_first);

namespace {

c10::optional<Tensor> some(const Tensor& t) {
  return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt;
}

// At the beginning of each backward pass.  A gradient that is itself to be
// differentiated would come out as a constant: refused.  So is one that is
// captured into a graph for a leaf whose gradients are summed on the default
// stream, since an eager graph of it lives: that stream would have to wait
// for the captured one, which ends the process.
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              ": the gradient is not differentiable (create_graph)");
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() ==
      c10::hip::CaptureStatus::None)
    return;
  const auto node = torch::autograd::get_current_node();
  for (size_t i = 0; node && i < node->num_outputs(); ++i) {
    const auto& leaf = node->next_edge(i).function;
    if (!leaf || leaf->num_outputs() != 0 ||
        !node->task_should_compute_output(i))
      continue;
    const auto on = leaf->stream();
    TORCH_CHECK(!on || on->id() != 0, what, ": a backward pass cannot be "
                "captured while an eager graph of the same leaves lives: "
                "delete its outputs first");
  }
}

// A matrix of the rows of x whose rows are contiguous.
Tensor matrix(const Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0,
              "rms_norm: x needs an axis with elements");
  Tensor m = x.numel() ? x.reshape({-1, x.size(-1)})
                       : x.new_empty({0, x.size(-1)});
  return m.stride(1) == 1 ? m : m.contiguous();
}

struct EmbedId : torch::autograd::Function<EmbedId> {
  static Tensor forward(AutogradContext* ctx, Tensor ids, Tensor w,
                        double scale, bool has_ignore, int64_t ignore) {
    ids = ids.contiguous();
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["has_ignore"] = has_ignore;
    ctx->saved_data["ignore"] = ignore;
    return embed_lookup(ids, w, scale, has_ignore, ignore);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("embed_id");
    Tensor gw;
    if (ctx->needs_input_grad(1))
      gw = embed_grad(ctx->get_saved_variables()[0], g[0].contiguous(),
                      ctx->saved_data["vocab"].toInt(),
                      ctx->saved_data["scale"].toDouble(),
                      ctx->saved_data["has_ignore"].toBool(),
                      ctx->saved_data["ignore"].toInt());
    return {Tensor(), gw, Tensor(), Tensor(), Tensor()};
  }
};

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor key,
                        int64_t threshold, double scale) {
    ctx->save_for_backward({key});
    ctx->saved_data["threshold"] = threshold;
    ctx->saved_data["scale"] = scale;
    return dropout(x.contiguous(), key, threshold, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("dropout");
    return {dropout(g[0].contiguous(), ctx->get_saved_variables()[0],
                    ctx->saved_data["threshold"].toInt(),
                    ctx->saved_data["scale"].toDouble()),
            Tensor(), Tensor(), Tensor()};
  }
};

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  // y, and the sum where there is a residual
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor w,
                               c10::optional<Tensor> res, double eps) {
    ctx->set_materialize_grads(false);
    if (res)
      TORCH_CHECK(res->sizes() == x.sizes(),
                  "rms_norm: the residual has another shape than x");
    w = w.contiguous();
    const Tensor m = matrix(x);
    const Tensor r = res ? matrix(*res) : Tensor();
    auto [y, h, rstd] = rms_norm_fwd(m, w, some(r), eps);
    ctx->save_for_backward({m, r, w, rstd});
    // not views, which could not be changed in place
    if (!res) return {at::_unsafe_view(y, x.sizes())};
    return {at::_unsafe_view(y, x.sizes()), at::_unsafe_view(h, x.sizes())};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("rms_norm");
    const auto s = ctx->get_saved_variables();
    const bool res = s[1].defined();
    const Tensor gh = res ? g[1] : Tensor();
    if (!g[0].defined())  // y was not used: the sum's gradient goes on
      return {gh, Tensor(), res ? gh : Tensor(), Tensor()};
    auto [dh, dw] = rms_norm_bwd(
        matrix(g[0]).contiguous(), s[0], some(s[1]),
        gh.defined() ? c10::optional<Tensor>(matrix(gh).contiguous())
                     : c10::nullopt,
        s[2], s[3]);
    dh = dh.view(g[0].sizes());
    return {dh, dw, res ? dh : Tensor(), Tensor()};
  }
};

struct LinearAttention : torch::autograd::Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, Tensor q, Tensor k,
                               Tensor v, Tensor log_decay,
                               c10::optional<Tensor> first,
                               c10::optional<Tensor> lengths, double scale) {
    ctx->set_materialize_grads(false);
    auto [o, last, states] =
        linear_attention_fwd(q, k, v, log_decay, first, lengths, scale);
    ctx->save_for_backward({q, k, v, log_decay,
                            first ? *first : Tensor(),
                            lengths ? *lengths : Tensor(), states});
    ctx->saved_data["scale"] = scale;
    return {o, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("linear_attention");
    const auto s = ctx->get_saved_variables();
    const Tensor none;
    if (!g[0].defined() && !g[1].defined())
      return {none, none, none, none, none, none, none};
    const Tensor go = g[0].defined() ? g[0] : at::zeros_like(s[2]);
    const bool need_first = s[4].defined() && ctx->needs_input_grad(4);
    auto [gq, gk, gv, gfirst] = linear_attention_bwd(
        s[0], s[1], s[2], s[3], some(s[4]), some(s[5]),
        ctx->saved_data["scale"].toDouble(), s[6], go,
        g[1].defined() ? c10::optional<Tensor>(g[1].contiguous())
                       : c10::nullopt,
        ctx->needs_input_grad(0), ctx->needs_input_grad(1),
        ctx->needs_input_grad(2), need_first);
    return {ctx->needs_input_grad(0) ? gq : none,
            ctx->needs_input_grad(1) ? gk : none,
            ctx->needs_input_grad(2) ? gv : none, none,
            need_first ? gfirst : none, none, none};
  }
};

}  // namespace

Tensor embed_id(Tensor ids, Tensor w, double scale, bool has_ignore,
                long ignore) {
  return EmbedId::apply(ids, w, scale, has_ignore, (int64_t)ignore);
}

Tensor dropout_fn(Tensor x, Tensor key, long threshold, double scale) {
  return Dropout::apply(x, key, (int64_t)threshold, scale);
}

variable_list rms_norm(Tensor x, Tensor w, c10::optional<Tensor> res,
                       double eps) {
  return RmsNorm::apply(x, w, res, eps);
}

variable_list linear_attention(Tensor q, Tensor k, Tensor v,
                               Tensor log_decay, c10::optional<Tensor> first,
                               c10::optional<Tensor> lengths, double scale) {
  return LinearAttention::apply(q, k, v, log_decay, first, lengths, scale);
}
