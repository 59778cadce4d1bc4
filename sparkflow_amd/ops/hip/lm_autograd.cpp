// Autograd nodes of the language-model operators, in C++: at the smallest
// sizes the kernels take a few microseconds, and a node in Python (its
// context, its backward under the interpreter lock on the engine's thread)
// would be most of a call.
#include <torch/extension.h>

#include <vector>

#include "lm_ops.h"

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

// Gradients that have no gradient of their own: a second derivative through
// them is an error, not a silent zero.
struct Once : public Function<Once> {
  static Tensor forward(AutogradContext*, Tensor grad, Tensor) {
    return grad.view_as(grad);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "this operator can be differentiated only once");
  }
};

// from: what the gradient was computed from.
Tensor once(const Tensor& grad, const variable_list& from) {
  if (!grad.defined() || !torch::GradMode::is_enabled()) return grad;
  for (const Tensor& t : from)
    if (t.defined() && t.requires_grad()) return Once::apply(grad, t);
  return grad;
}

// The kernels below see tensors without history.
struct NoGrad {
  torch::AutoGradMode mode{false};
};

c10::optional<Tensor> given(const Tensor& t) {
  if (!t.defined()) return c10::nullopt;
  return t;
}

struct Dropout : public Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor state,
                        int64_t keep, double scale) {
    ctx->save_for_backward({state});
    ctx->saved_data["keep"] = keep;
    ctx->saved_data["scale"] = scale;
    if (keep == 0)
      return torch::zeros_like(x, x.options(), at::MemoryFormat::Contiguous);
    return dropout(x.contiguous(), state, keep, scale);
  }
  // linear in x with the same mask, and differentiable again by itself
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return {Dropout::apply(g[0], ctx->get_saved_variables()[0],
                           ctx->saved_data["keep"].toInt(),
                           ctx->saved_data["scale"].toDouble()),
            Tensor(), Tensor(), Tensor()};
  }
};

struct Logprobs : public Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, Tensor logits,
                               Tensor tokens, int64_t k, int64_t ignore) {
    ctx->set_materialize_grads(false);
    const auto r = logprobs_fwd(logits, tokens, k, ignore);
    const Tensor &logp = r[0], &entropy = r[1], &top = r[3], &ids = r[4];
    ctx->save_for_backward({logits, tokens, r[2], entropy, ids});
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({ids});
    return {logp, entropy, top, ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    Tensor dx;
    {
      NoGrad none;
      for (int i = 0; i < 3; ++i)
        if (g[i].defined()) g[i] = g[i].contiguous();
      dx = logprobs_bwd(s[0], s[1], s[2], s[3], s[4], given(g[0]),
                        given(g[1]), given(g[2]),
                        ctx->saved_data["ignore"].toInt());
    }
    return {once(dx, {s[0], g[0], g[1], g[2]}), Tensor(), Tensor(),
            Tensor()};
  }
};

struct AdapterAdd : public Function<AdapterAdd> {
  static Tensor forward(AutogradContext* ctx, Tensor base, Tensor x, Tensor a,
                        Tensor b, c10::optional<Tensor> scales, Tensor ids,
                        Tensor plan, double scale, int64_t act) {
    const Tensor z =
        adapter_shrink(x, a, ids, plan, scales, scale, true, false);
    const Tensor y = adapter_expand(base, z, b, ids, plan, act, true);
    ctx->save_for_backward(
        {x, a, b, z, scales.has_value() ? *scales : Tensor(), ids, plan,
         act ? y : Tensor()});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &a = s[1], &b = s[2], &z = s[3], &ids = s[5],
                 &plan = s[6];
    const int64_t E = a.size(0), R = a.size(1);
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool need_x = ctx->needs_input_grad(1);
    const bool need_a = ctx->needs_input_grad(2);
    const bool need_b = ctx->needs_input_grad(3);
    Tensor dy, dx, da, db;
    {
      NoGrad none;
      dy = g[0].contiguous();
      if (act) dy = adapter_act_bwd(s[7], dy, act);
      Tensor dz;
      if (need_x || need_a)
        dz = adapter_shrink(dy, b, ids, plan, given(s[4]),
                            ctx->saved_data["scale"].toDouble(), false, false);
      if (need_x)
        dx = adapter_expand(c10::nullopt, dz, a, ids, plan, 0, false);
      if (need_a || need_b) {
        const auto none = c10::optional<Tensor>();
        const auto d = adapter_outer(
            need_a ? given(x) : none, need_a ? given(dz) : none,
            need_b ? given(dy) : none, need_b ? given(z) : none, ids, plan, E,
            R);
        da = d[0];
        db = d[1];
      }
    }
    const variable_list from = {g[0], x, a, b};
    Tensor dbase;
    if (ctx->needs_input_grad(0))
      dbase = act ? once(dy, {g[0], s[7]}) : g[0];
    return {dbase,    once(dx, from), once(da, from), once(db, from),
            Tensor(), Tensor(),       Tensor(),       Tensor(),
            Tensor()};
  }
};

// Rows of `width` side by side; a view where the layout allows.
Tensor rows_of(const Tensor& t, int64_t width) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  return width == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

}  // namespace

Tensor dropout_apply(Tensor x, Tensor state, int64_t keep, double scale) {
  return Dropout::apply(x, state, keep, scale);
}

std::vector<Tensor> logprobs_apply(Tensor logits, Tensor tokens, int64_t k,
                                   int64_t ignore) {
  const auto shape = tokens.sizes().vec();
  Tensor t = tokens.dim() == 1 ? tokens : tokens.reshape(-1);
  auto r = Logprobs::apply(rows_of(logits, logits.size(-1)), t.contiguous(),
                           k, ignore);
  if (tokens.dim() != 1) {
    auto tops = shape;
    tops.push_back(k);
    for (int i = 0; i < 4; ++i) r[i] = r[i].reshape(i < 2 ? shape : tops);
  }
  return r;
}

// plan: what adapter_plan gave for ids, or none.
Tensor adapter_add_apply(Tensor base, Tensor x, Tensor a, Tensor b,
                         c10::optional<Tensor> scales, double scale,
                         Tensor ids, c10::optional<Tensor> plan,
                         int64_t act) {
  const Tensor rows = ids.reshape(-1).contiguous();
  const Tensor base2 = rows_of(base, b.size(1)), x2 = rows_of(x, a.size(2));
  const Tensor a2 = a.contiguous(), b2 = b.contiguous();
  const Tensor p = plan.has_value() ? *plan : adapter_plan(rows, a.size(0));
  Tensor y;
  if (torch::GradMode::is_enabled() &&
      (base.requires_grad() || x.requires_grad() || a.requires_grad() ||
       b.requires_grad())) {
    y = AdapterAdd::apply(base2, x2, a2, b2, scales, rows, p, scale, act);
  } else {
    const Tensor z =
        adapter_shrink(x2, a2, rows, p, scales, scale, true, true);
    y = adapter_expand(base2, z, b2, rows, p, act, true);
  }
  return base.dim() == 2 ? y : y.reshape(base.sizes());
}
