// Autograd nodes of the native layer normalisation, in C++: for a batch of a few thousand
// rows the kernels take 10 to 50 us, and two nodes written in Python cost twice that.
#include <torch/extension.h>

namespace pb {

std::vector<at::Tensor> add_layernorm_fwd(at::Tensor x, c10::optional<at::Tensor> delta, at::Tensor w,
                                          c10::optional<at::Tensor> b, double eps, bool out_bf16, bool stats);
at::Tensor layernorm_bwd(at::Tensor dy, at::Tensor x, at::Tensor w, at::Tensor mean, at::Tensor rstd,
                         c10::optional<at::Tensor> dres, c10::optional<at::Tensor> dx_bf16, at::Tensor dw_out,
                         c10::optional<at::Tensor> db_out, bool accumulate);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Contiguous rows of the last dimension.
at::Tensor rows_of(const at::Tensor& t, int64_t n) {
  if (t.dim() == 2 && t.is_contiguous()) return t;
  return t.reshape({-1, n}).contiguous();
}
// A result in its caller's shape.  Not a view for autograd: torch refuses to change a view that a
// node returned in place.
at::Tensor shaped(const at::Tensor& t, const at::Tensor& like) {
  return t.dim() == like.dim() ? t : at::_unsafe_view(t, like.sizes());
}
at::Tensor param_of(const at::Tensor& w) { return w.to(at::kFloat).contiguous(); }
c10::optional<at::Tensor> param_of(const c10::optional<at::Tensor>& b) {
  return b.has_value() ? c10::optional<at::Tensor>(param_of(*b)) : c10::nullopt;
}
// Tangents of forward-mode differentiation would be dropped: the kernels work on raw memory, and
// whether a node is made depends on the backward pass alone.
void refuse_tangent(const at::Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "layernorm: forward-mode derivatives are not available on CUDA");
}
void refuse_tangent(const c10::optional<at::Tensor>& t) {
  if (t.has_value()) refuse_tangent(*t);
}
bool wants_grad(const at::Tensor& t) { return t.requires_grad(); }
bool wants_grad(const c10::optional<at::Tensor>& t) { return t.has_value() && t->requires_grad(); }

struct Grads {
  at::Tensor dx, dw, db;
};
Grads backward_rows(AutogradContext* ctx, const at::Tensor& dy, c10::optional<at::Tensor> dres,
                    c10::optional<at::Tensor> dx_bf16) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "layernorm: its backward pass is not differentiable (create_graph)");
  const auto saved = ctx->get_saved_variables();
  const at::Tensor x = rows_of(saved[0], saved[0].size(-1)), &w = saved[1];
  auto dw = at::empty({x.size(1)}, x.options().dtype(at::kFloat));
  c10::optional<at::Tensor> db;
  const int64_t bias_type = ctx->saved_data["bias_type"].toInt();
  if (bias_type >= 0) db = at::empty_like(dw);
  auto dx = layernorm_bwd(rows_of(dy, x.size(1)), x, param_of(w), saved[2], saved[3], dres, dx_bf16, dw, db, false);
  return {dx, dw.to(w.scalar_type()), db.has_value() ? db->to(static_cast<at::ScalarType>(bias_type)) : at::Tensor()};
}
void save(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& b,
          const at::Tensor& mean, const at::Tensor& rstd) {
  ctx->save_for_backward({x, w, mean, rstd});
  ctx->saved_data["bias_type"] = b.has_value() ? static_cast<int64_t>(b->scalar_type()) : int64_t(-1);
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const c10::optional<at::Tensor>& b, double eps) {
    auto x2 = rows_of(x, x.size(-1));
    auto r = add_layernorm_fwd(x2, c10::nullopt, param_of(w), param_of(b), eps, false, true);
    save(ctx, x2, w, b, r[2], r[3]);
    return shaped(r[1], x);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor& dy = grads[0];
    auto g = backward_rows(ctx, dy, c10::nullopt, c10::nullopt);
    return {g.dx.view(dy.sizes()), g.dw, g.db, at::Tensor()};
  }
};

struct AddLayerNormFn : torch::autograd::Function<AddLayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& delta, const at::Tensor& w,
                               const c10::optional<at::Tensor>& b, double eps) {
    const int64_t n = x.size(-1);
    auto r = add_layernorm_fwd(rows_of(x, n), rows_of(delta, n), param_of(w), param_of(b), eps, true, true);
    // saved as it is returned, so that a change in place is noticed by the backward pass
    auto total = shaped(r[0], x);
    save(ctx, total, w, b, r[2], r[3]);
    return {total, shaped(r[1], x)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor &dtotal = grads[0], &dy = grads[1];
    const int64_t n = dy.size(-1);
    auto ddelta = at::empty({dy.numel() / n, n}, dy.options().dtype(at::kBFloat16));
    auto g = backward_rows(ctx, dy, rows_of(dtotal, n), ddelta);
    return {g.dx.view(dy.sizes()), ddelta.view(dy.sizes()), g.dw, g.db, at::Tensor()};
  }
};

}  // namespace

// Public forms (arguments already checked): a node only where a gradient is wanted.
at::Tensor layernorm(at::Tensor x, at::Tensor w, c10::optional<at::Tensor> b, double eps) {
  refuse_tangent(x);
  refuse_tangent(w);
  refuse_tangent(b);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b)))
    return LayerNormFn::apply(x, w, b, eps);
  at::NoGradGuard guard;
  return shaped(add_layernorm_fwd(rows_of(x, x.size(-1)), c10::nullopt, param_of(w), param_of(b), eps, false, false)[1],
                x);
}

std::vector<at::Tensor> add_layernorm(at::Tensor x, at::Tensor delta, at::Tensor w, c10::optional<at::Tensor> b,
                                      double eps) {
  refuse_tangent(x);
  refuse_tangent(delta);
  refuse_tangent(w);
  refuse_tangent(b);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(delta) || wants_grad(w) || wants_grad(b)))
    return AddLayerNormFn::apply(x, delta, w, b, eps);
  at::NoGradGuard guard;
  const int64_t n = x.size(-1);
  auto r = add_layernorm_fwd(rows_of(x, n), rows_of(delta, n), param_of(w), param_of(b), eps, true, false);
  return {shaped(r[0], x), shaped(r[1], x)};
}

}  // namespace pb
