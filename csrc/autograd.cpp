// Autograd nodes of the vocabulary operators (embedding.cu, linear_ce.cu, distill.cu).
// They are recorded and run without the interpreter: for the small calls of these
// operators a Python-level node costs more than the kernels (256 tokens of 64 fp16
// columns, forward and gradient: 87 us with Python nodes).
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <initializer_list>
#include <memory>
#include <tuple>

namespace lrb {

at::Tensor embedding_fwd(const at::Tensor&, const at::Tensor&, double);
at::Tensor embedding_bwd(const at::Tensor&, const at::Tensor&, int64_t, int64_t, double);
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> linear_ce_fwd(const at::Tensor&, const at::Tensor&,
                                                                         const at::Tensor&, int64_t, int64_t);
std::tuple<at::Tensor, at::Tensor> linear_ce_bwd(const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t,
                                                 const at::Tensor&, const at::Tensor&, bool, const at::Tensor&, int64_t,
                                                 bool, bool);
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> distill_fwd(const at::Tensor&,
                                                                                   const at::Tensor&,
                                                                                   const at::Tensor&, double, int64_t,
                                                                                   bool);
at::Tensor distill_bwd(const at::Tensor&, const at::Tensor&, double, const at::Tensor&, const at::Tensor&,
                       const at::Tensor&, bool, const at::Tensor&);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Gradients that have no gradient of their own: differentiating them raises.
variable_list once(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once",
                                                             (int64_t)grads.size());
  return (*err)(std::move(grads));
}

at::Tensor unit_columns(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); }

// Forward mode: the kernels see values only, so a tangent is followed (the lookup, which
// is linear) or refused.  Detached values have none.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }

void refuse_tangents(const char* name, std::initializer_list<at::Tensor> inputs) {
  for (const auto& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), name, " has no forward-mode derivative");
}

bool tracked(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// scale * w[ids], and the gradient of w, with their derivatives of both modes.
at::Tensor lookup(const at::Tensor& w, const at::Tensor& ids, double scale, int64_t padding);
at::Tensor table_gradient(const at::Tensor& dy, const at::Tensor& ids, int64_t rows, double scale, int64_t padding);

struct EmbeddingFn : public Function<EmbeddingFn> {
  static Variable forward(AutogradContext* ctx, const Variable& w, const Variable& ids, double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embedding_fwd(ids, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g);
};

// The gradient is linear in dy; its own gradient is the lookup (zero at the padding
// token and at ids outside the table).
struct EmbeddingGradFn : public Function<EmbeddingGradFn> {
  static Variable forward(AutogradContext* ctx, const Variable& dy, const Variable& ids, int64_t rows, double scale,
                          int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = rows;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embedding_bwd(unit_columns(dy), ids, rows, padding, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto ids = ctx->get_saved_variables()[0];
    const int64_t padding = ctx->saved_data["padding"].toInt();
    const auto out = lookup(g[0], ids, ctx->saved_data["scale"].toDouble(), padding);
    const auto kept = ids.ge(0).logical_and(ids.lt(ctx->saved_data["rows"].toInt())).logical_and(ids.ne(padding));
    return {at::where(kept.unsqueeze(1), out, at::zeros({}, out.options())), Variable(), Variable(), Variable(),
            Variable()};
  }
};

variable_list EmbeddingFn::backward(AutogradContext* ctx, variable_list g) {
  const auto ids = ctx->get_saved_variables()[0];
  return {table_gradient(g[0], ids, ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(),
                         ctx->saved_data["padding"].toInt()),
          Variable(), Variable(), Variable()};
}

at::Tensor lookup(const at::Tensor& w, const at::Tensor& ids, double scale, int64_t padding) {
  if (has_tangent(w)) {
    const auto [value, tangent] = at::_unpack_dual(w, 0);
    return at::_make_dual(lookup(value, ids, scale, padding), lookup(tangent, ids, scale, padding), 0);
  }
  const at::Tensor table = unit_columns(w);
  return tracked(table) ? EmbeddingFn::apply(table, ids, scale, padding) : embedding_fwd(ids, table, scale);
}

at::Tensor table_gradient(const at::Tensor& dy, const at::Tensor& ids, int64_t rows, double scale, int64_t padding) {
  if (has_tangent(dy)) {
    const auto [value, tangent] = at::_unpack_dual(dy, 0);
    return at::_make_dual(table_gradient(value, ids, rows, scale, padding),
                          table_gradient(tangent, ids, rows, scale, padding), 0);
  }
  return at::GradMode::is_enabled() ? EmbeddingGradFn::apply(dy, ids, rows, scale, padding)
                                    : embedding_bwd(unit_columns(dy), ids, rows, padding, scale);
}

struct LinearCEFn : public Function<LinearCEFn> {
  static Variable forward(AutogradContext* ctx, const Variable& h, const Variable& w, const Variable& targets,
                          int64_t ignore, int64_t reduction, int64_t piece) {
    auto [rows, stats, out, factor] = linear_ce_fwd(h, w, targets, ignore, reduction);
    ctx->save_for_backward({h, w, targets, stats, factor});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["per_row"] = reduction == 0;
    ctx->saved_data["piece"] = piece;
    return reduction == 0 ? rows : out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    refuse_tangents("piecewise_linear_cross_entropy", {g[0]});
    const auto s = ctx->get_saved_variables();
    const bool per_row = ctx->saved_data["per_row"].toBool(), need_h = ctx->needs_input_grad(0),
               need_w = ctx->needs_input_grad(1);
    at::Tensor dh, dw;
    {
      at::AutoGradMode off(false);
      std::tie(dh, dw) = linear_ce_bwd(s[0], s[1], s[2], ctx->saved_data["ignore"].toInt(), s[3],
                                       g[0].to(at::kFloat).contiguous(), per_row,
                                       per_row ? s[3] : s[4], ctx->saved_data["piece"].toInt(), need_h,
                                       need_w);
    }
    return once("piecewise_linear_cross_entropy", {need_h ? dh : Variable(), need_w ? dw : Variable(), Variable(),
                                                   Variable(), Variable(), Variable()});
  }
};

struct DistillFn : public Function<DistillFn> {
  static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& teacher, const Variable& ids,
                          double temperature, int64_t reduction) {
    auto [rows, stats, probs, out, factor] = distill_fwd(x, teacher, ids, temperature, reduction, true);
    ctx->save_for_backward({x, ids, stats, probs, factor});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["per_row"] = reduction == 0;
    return reduction == 0 ? rows : out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    refuse_tangents("topk_distillation", {g[0]});
    const auto s = ctx->get_saved_variables();
    const bool per_row = ctx->saved_data["per_row"].toBool();
    at::Tensor dx;
    {
      at::AutoGradMode off(false);
      dx = distill_bwd(s[0], s[1], ctx->saved_data["temperature"].toDouble(), s[2], s[3],
                       g[0].to(at::kFloat).contiguous(), per_row, per_row ? s[2] : s[4]);
    }
    return once("topk_distillation", {dx, Variable(), Variable(), Variable(), Variable()});
  }
};

}  // namespace

// `ids` of any shape and strides; out (*ids.shape, d).
at::Tensor embedding(const at::Tensor& ids, const at::Tensor& w, double scale, int64_t padding) {
  const at::Tensor flat = (ids.dim() == 1 ? ids : ids.reshape({-1})).contiguous();
  const at::Tensor out = lookup(w, flat, scale, padding);
  if (ids.dim() == 1) return out;
  auto shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  return out.view(shape);
}

// h (..., d), targets of its leading shape; a row loss for each target with reduction 0.
at::Tensor piecewise_linear_ce(const at::Tensor& h, const at::Tensor& w, const at::Tensor& targets, int64_t ignore,
                               int64_t reduction, int64_t piece) {
  refuse_tangents("piecewise_linear_cross_entropy", {h, w});
  const auto rows16 = [](const at::Tensor& t) {  // rows that the tensor maps take: 16-byte aligned, unit columns
    return t.stride(1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                   t.stride(0) * (int64_t)t.element_size() % 16 == 0 && (t.stride(0) >= t.size(1) || t.size(0) <= 1)
               ? t
               : t.clone(at::MemoryFormat::Contiguous);  // a contiguous tensor may start anywhere
  };
  const at::Tensor h2 = rows16(h.dim() == 2 ? h : h.reshape({targets.numel(), w.size(1)})), w2 = rows16(w),
                   t = (targets.dim() == 1 ? targets : targets.reshape({-1})).contiguous();
  at::Tensor loss;
  if (tracked(h2) || tracked(w2)) {
    loss = LinearCEFn::apply(h2, w2, t, ignore, reduction, piece);
  } else {
    auto [rows, stats, out, factor] = linear_ce_fwd(h2, w2, t, ignore, reduction);
    loss = reduction == 0 ? rows : out;
  }
  return reduction == 0 && targets.dim() != 1 ? loss.view(targets.sizes()) : loss;
}

// x (..., V); teacher and ids (..., K).  (B, S, V) views with any strides of the leading
// dimensions are read in place.
at::Tensor topk_distillation(const at::Tensor& x, const at::Tensor& teacher, const at::Tensor& ids, double temperature,
                             int64_t reduction) {
  refuse_tangents("topk_distillation", {x});
  const int64_t V = x.size(-1), K = ids.size(-1);
  const at::Tensor x3 = unit_columns(x.dim() == 3 ? x : x.dim() == 2 ? x.unsqueeze(0) : x.reshape({1, -1, V}));
  const at::Tensor t2 = (teacher.dim() == 2 ? teacher : teacher.reshape({-1, K})).detach().contiguous(),
                   i2 = (ids.dim() == 2 ? ids : ids.reshape({-1, K})).contiguous();
  at::Tensor loss;
  if (tracked(x3)) {
    loss = DistillFn::apply(x3, t2, i2, temperature, reduction);
  } else {
    auto [rows, stats, probs, out, factor] = distill_fwd(x3, t2, i2, temperature, reduction, false);
    loss = reduction == 0 ? rows : out;
  }
  return reduction == 0 && x.dim() != 2 ? loss.view(x.sizes().slice(0, x.dim() - 1)) : loss;
}

}  // namespace lrb
