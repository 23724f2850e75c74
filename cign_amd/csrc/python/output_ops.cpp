// The operators at the model's output as autograd nodes of their own: LayerNorm
// of any width, the log probabilities of rows of logits, the loss against a
// teacher's list. Host code only: allocations from torch's caching allocator,
// the current stream and device, and the C-ABI's calls.
//
// In C++ and not as Python autograd functions because a training step's
// backward runs on the engine's own thread: there a Python function takes the
// interpreter from the main thread with its caches cold (a call with its
// gradient of rows that take the GPU 6 to 30 us: 90 to 120 us).
//
// Each is an operator of torch's dispatcher (cign_amd::layernorm, ...), and so are the
// passes with the statistics a gradient takes and the gradients: a trace, or
// another mode that records operators, records the calls and not the allocations
// in them, and transforms that have no rule for them refuse. The autograd key's
// kernel applies the node where a gradient is needed or an input has a
// forward-mode derivative, which the node refuses. A trace repeats a call without the
// checks of the Python functions, with other shapes if it likes, so what a
// kernel's accesses rest on is checked here.
//
// The gradients are once differentiable: what a graph of the gradient would
// hold is an error, as once_differentiable makes it.
#include "ops.h"

namespace {

using namespace cign_ops;

constexpr int64_t kStats = 8;  // floats a row that the distillation's backward reads

// ---- LayerNorm -------------------------------------------------------------

Tensor run_layernorm(const Tensor& x, const Optional& weight_, const Optional& bias_, double eps, Tensor* stats) {
  check_rows(x, "x");
  const int64_t n = row_count(x), D = x.size(-1);
  const Tensor weight = whole(weight_), bias = whole(bias_);
  const Tensor& param = weight.defined() ? weight : bias.defined() ? bias : x;
  TORCH_CHECK_TYPE(param.scalar_type() == at::kFloat || param.scalar_type() == x.scalar_type(),
                   "LayerNorm weight/bias must both be float32 or both of x's type");
  if (weight.defined()) check_beside(weight, x, "LayerNorm weight", param.scalar_type(), {D});
  if (bias.defined()) check_beside(bias, x, "LayerNorm bias", param.scalar_type(), {D});
  const Tensor y = like(x, x.sizes(), x.scalar_type());
  if (stats) *stats = like(x, {2, n}, at::kFloat);
  if (x.is_meta()) return y;
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  float* mean = stats ? stats->data_ptr<float>() : nullptr;
  check(cign_layernorm_fwd(stream_of(x), n, static_cast<int32_t>(D), code(x.scalar_type()), code(param.scalar_type()),
                           rows.data_ptr(), rows.stride(0), ptr(weight), ptr(bias), static_cast<float>(eps),
                           y.data_ptr(), mean, mean ? mean + n : nullptr),
        "cign_layernorm_fwd");
  return y;
}

Tensor layernorm(const Tensor& x, const Optional& weight, const Optional& bias, double eps) {
  return run_layernorm(x, weight, bias, eps, nullptr);
}

// y and the rows' mean and 1 / sqrt(var + eps)
std::tuple<Tensor, Tensor> layernorm_forward(const Tensor& x, const Optional& weight, const Optional& bias,
                                             double eps) {
  Tensor stats;
  Tensor y = run_layernorm(x, weight, bias, eps, &stats);
  return {y, stats};
}

// the gradients asked for of (x, weight, bias), the parameters' in `type`
variable_list layernorm_backward(const Tensor& grad, const Tensor& x, const Optional& weight_, const Tensor& stats,
                                 at::ScalarType type, bool of_x, bool of_weight, bool of_bias) {
  check_rows(x, "x");
  const int64_t n = row_count(x), D = x.size(-1);
  const Tensor weight = whole(weight_);
  TORCH_CHECK_TYPE(type == at::kFloat || type == x.scalar_type(), "the parameters are float32 or of x's type");
  check_beside(grad, x, "the gradient", x.scalar_type(), x.sizes());
  check_beside(stats, x, "the statistics", at::kFloat, {2, n});
  if (weight.defined()) check_beside(weight, x, "LayerNorm weight", type, {D});
  Tensor gx, gw, gb;
  variable_list out;
  if (of_x) out.push_back(gx = like(x, x.sizes(), x.scalar_type()));
  if (of_weight) out.push_back(gw = like(x, {D}, type));
  if (of_bias) out.push_back(gb = like(x, {D}, type));
  if (x.is_meta()) return out;
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x), gy = as_rows(grad), kept = stats.contiguous();
  const int64_t bytes =
      of_weight || of_bias ? cign_layernorm_bwd_workspace_bytes(n, static_cast<int32_t>(D)) : 0;
  const Tensor ws = workspace(x, bytes);
  const float* mean = kept.data_ptr<float>();
  check(cign_layernorm_bwd(stream_of(x), n, static_cast<int32_t>(D), code(x.scalar_type()), code(type), gy.data_ptr(),
                           gy.stride(0), rows.data_ptr(), rows.stride(0), ptr(weight), mean, mean + n, ptr(gx), ptr(gw),
                           ptr(gb), ptr(ws), bytes),
        "cign_layernorm_bwd");
  return out;
}

CIGN_OP(layernorm, layernorm)
CIGN_OP(layernorm_forward, layernorm_forward)
CIGN_OP(layernorm_backward, layernorm_backward)

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Optional& weight, const Optional& bias, double eps,
                        bool graph) {
    const at::AutoDispatchBelowADInplaceOrView below;
    if (!graph) return call_layernorm(x, weight, bias, eps);
    auto [y, stats] = call_layernorm_forward(x, weight, bias, eps);
    ctx->save_for_backward({x, value(weight), stats});
    ctx->saved_data["params"] =
        static_cast<int64_t>(weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type());
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& weight = saved[1];
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      // the edges count the tensors that were given
      const bool of[3] = {ctx->needs_input_grad(0), weight.defined() && ctx->needs_input_grad(1),
                          ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1)};
      const variable_list given =
          call_layernorm_backward(grads[0], saved[0], optional(weight), saved[2],
                                  static_cast<at::ScalarType>(ctx->saved_data["params"].toInt()), of[0], of[1], of[2]);
      for (size_t i = 0, k = 0; i < 3; ++i)
        if (of[i]) out[i] = given[k++];
    }
    return sealed(std::move(out), "fused_layernorm");
  }
};

Tensor layernorm_autograd(const Tensor& x, const Optional& weight, const Optional& bias, double eps) {
  const bool graph = at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) ||
                                                    (bias && bias->requires_grad()));
  if (!graph && !has_tangent(x) && !has_tangent(weight) && !has_tangent(bias)) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_layernorm(x, weight, bias, eps);
  }
  return LayerNorm::apply(x, optional(whole(weight)), optional(whole(bias)), eps, graph);
}

// ---- log probabilities -------------------------------------------------------

// entropy, then logprob with labels, then top log probabilities and indices with top_k
variable_list run_logprobs(const Tensor& x, const Optional& labels_, int64_t top_k, double temperature,
                           int64_t ignore_index, Tensor* stats) {
  check_rows(x, "logits");
  const int64_t n = row_count(x);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= x.size(-1), "top_k must be in [0, V], got ", top_k, " for V = ", x.size(-1));
  const Tensor labels = whole(labels_);
  if (labels.defined()) check_beside(labels, x, "labels", at::kLong, lead(x));
  variable_list out{like(x, lead(x), at::kFloat)};
  Tensor logprob, top, index;
  if (labels.defined()) out.push_back(logprob = like(x, lead(x), at::kFloat));
  if (top_k) {
    std::vector<int64_t> shape = lead(x).vec();
    shape.push_back(top_k);
    out.push_back(top = like(x, shape, at::kFloat));
    out.push_back(index = like(x, shape, at::kLong));
  }
  if (stats) *stats = like(x, {n, 4}, at::kFloat);
  if (x.is_meta()) return out;
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  const int32_t V = static_cast<int32_t>(x.size(-1)), K = static_cast<int32_t>(top_k), type = code(x.scalar_type());
  const int64_t bytes = cign_class_logprobs_workspace_bytes(type, n, V, K);
  const Tensor ws = workspace(x, bytes);
  check(cign_class_logprobs_fwd(stream_of(x), type, n, V, rows.data_ptr(), rows.stride(0),
                                static_cast<float>(temperature), ptr<int64_t>(labels), ignore_index, K,
                                ptr<float>(logprob), out[0].data_ptr<float>(), ptr<float>(top), ptr<int64_t>(index),
                                stats ? stats->data_ptr<float>() : nullptr, ptr(ws), bytes),
        "cign_class_logprobs_fwd");
  return out;
}

variable_list class_logprobs(const Tensor& x, const Optional& labels, int64_t top_k, double temperature,
                             int64_t ignore_index) {
  return run_logprobs(x, labels, top_k, temperature, ignore_index, nullptr);
}

// the same and, last, the rows' statistics
variable_list class_logprobs_forward(const Tensor& x, const Optional& labels, int64_t top_k, double temperature,
                                     int64_t ignore_index) {
  Tensor stats;
  variable_list out = run_logprobs(x, labels, top_k, temperature, ignore_index, &stats);
  out.push_back(stats);
  return out;
}

Tensor class_logprobs_backward(const Optional& grad_entropy, const Optional& grad_logprob, const Tensor& x,
                               const Optional& labels_, const Tensor& stats, double temperature, int64_t ignore_index) {
  check_rows(x, "logits");
  const int64_t n = row_count(x);
  const Tensor labels = whole(labels_), ge = whole(grad_entropy), gl = whole(grad_logprob);
  check_beside(stats, x, "the statistics", at::kFloat, {n, 4});
  if (labels.defined()) check_beside(labels, x, "labels", at::kLong, lead(x));
  if (ge.defined()) check_beside(ge, x, "the entropy's gradient", at::kFloat, lead(x));
  if (gl.defined()) check_beside(gl, x, "the log probabilities' gradient", at::kFloat, lead(x));
  Tensor gx = like(x, x.sizes(), x.scalar_type());
  if (x.is_meta()) return gx;
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x), kept = stats.contiguous();
  check(cign_class_logprobs_bwd(stream_of(x), code(x.scalar_type()), n, static_cast<int32_t>(x.size(-1)),
                                rows.data_ptr(), rows.stride(0), static_cast<float>(temperature), ptr<int64_t>(labels),
                                ignore_index, kept.data_ptr<float>(), ptr<float>(gl), ptr<float>(ge), gx.data_ptr()),
        "cign_class_logprobs_bwd");
  return gx;
}

CIGN_OP(class_logprobs, class_logprobs)
CIGN_OP(class_logprobs_forward, class_logprobs_forward)
CIGN_OP(class_logprobs_backward, class_logprobs_backward)

struct Logprobs : torch::autograd::Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Optional& labels, int64_t top_k,
                               double temperature, int64_t ignore_index, bool graph) {
    const at::AutoDispatchBelowADInplaceOrView below;
    if (!graph) return call_class_logprobs(x, labels, top_k, temperature, ignore_index);
    variable_list out = call_class_logprobs_forward(x, labels, top_k, temperature, ignore_index);
    ctx->save_for_backward({x, value(labels), out.back()});
    out.pop_back();
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore_index;
    ctx->set_materialize_grads(false);
    if (top_k) ctx->mark_non_differentiable({out[out.size() - 2], out.back()});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& labels = saved[1];
    variable_list out(6);
    const Tensor given = labels.defined() ? grads[1] : Tensor();
    if (!grads[0].defined() && !given.defined()) return out;
    {
      const at::NoGradGuard no_grad;
      out[0] = call_class_logprobs_backward(optional(grads[0]), optional(given), saved[0], optional(labels), saved[2],
                                            ctx->saved_data["temperature"].toDouble(),
                                            ctx->saved_data["ignore"].toInt());
    }
    return sealed(std::move(out), "class_logprobs");
  }
};

variable_list class_logprobs_autograd(const Tensor& x, const Optional& labels, int64_t top_k, double temperature,
                                      int64_t ignore_index) {
  const bool graph = at::GradMode::is_enabled() && x.requires_grad();
  if (!graph && !has_tangent(x)) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_class_logprobs(x, labels, top_k, temperature, ignore_index);
  }
  return Logprobs::apply(x, labels, top_k, temperature, ignore_index, graph);
}

// ---- distillation ------------------------------------------------------------

Tensor run_distill(const Tensor& x, const Tensor& teacher_, const Tensor& index_, double temperature, bool tail,
                   Tensor* kept) {
  check_rows(x, "logits");
  TORCH_CHECK_VALUE(index_.dim() >= 1, "teacher_index must be [..., K], got ", index_.sizes());
  const int64_t n = row_count(x), K = index_.size(-1);
  std::vector<int64_t> shape = lead(x).vec();
  shape.push_back(K);
  check_beside(teacher_, x, "teacher_logprobs", at::kFloat, shape);
  check_beside(index_, x, "teacher_index", at::kLong, shape);
  TORCH_CHECK_VALUE(K <= std::numeric_limits<int32_t>::max(), "too long a list");
  Tensor loss = like(x, lead(x), at::kFloat);
  if (kept) *kept = like(x, {n * (kStats + K)}, at::kFloat);  // the rows' statistics, then their lists' masses
  if (x.is_meta()) return loss;
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x), teacher = teacher_.contiguous(), index = index_.contiguous();
  const int32_t V = static_cast<int32_t>(x.size(-1)), type = code(x.scalar_type());
  float* stats = kept ? kept->data_ptr<float>() : nullptr;
  const int64_t bytes = cign_distill_topk_workspace_bytes(type, n, V);
  const Tensor ws = workspace(x, bytes);
  check(cign_distill_topk_fwd(stream_of(x), type, n, V, rows.data_ptr(), rows.stride(0),
                              static_cast<float>(temperature), tail, static_cast<int32_t>(K),
                              teacher.data_ptr<float>(), index.data_ptr<int64_t>(), loss.data_ptr<float>(), stats,
                              stats ? stats + n * kStats : nullptr, ptr(ws), bytes),
        "cign_distill_topk_fwd");
  return loss;
}

Tensor distill_topk(const Tensor& x, const Tensor& teacher, const Tensor& index, double temperature, bool tail) {
  return run_distill(x, teacher, index, temperature, tail, nullptr);
}

// the loss and what its gradient takes
std::tuple<Tensor, Tensor> distill_topk_forward(const Tensor& x, const Tensor& teacher, const Tensor& index,
                                                double temperature, bool tail) {
  Tensor kept;
  Tensor loss = run_distill(x, teacher, index, temperature, tail, &kept);
  return {loss, kept};
}

Tensor distill_topk_backward(const Tensor& grad, const Tensor& x, const Tensor& index_, const Tensor& kept_,
                             double temperature) {
  check_rows(x, "logits");
  TORCH_CHECK_VALUE(index_.dim() >= 1, "teacher_index must be [..., K], got ", index_.sizes());
  const int64_t n = row_count(x), K = index_.size(-1);
  std::vector<int64_t> shape = lead(x).vec();
  shape.push_back(K);
  check_beside(index_, x, "teacher_index", at::kLong, shape);
  TORCH_CHECK_VALUE(K <= std::numeric_limits<int32_t>::max(), "too long a list");
  check_beside(kept_, x, "the statistics", at::kFloat, {n * (kStats + K)});
  check_beside(grad, x, "the loss's gradient", at::kFloat, lead(x));
  Tensor gx = like(x, x.sizes(), x.scalar_type());
  if (x.is_meta()) return gx;
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x), g = grad.contiguous(), index = index_.contiguous(), kept = kept_.contiguous();
  const float* stats = kept.data_ptr<float>();
  check(cign_distill_topk_bwd(stream_of(x), code(x.scalar_type()), n, static_cast<int32_t>(x.size(-1)),
                              rows.data_ptr(), rows.stride(0), static_cast<float>(temperature),
                              static_cast<int32_t>(K), index.data_ptr<int64_t>(), stats, stats + n * kStats,
                              g.data_ptr<float>(), gx.data_ptr()),
        "cign_distill_topk_bwd");
  return gx;
}

CIGN_OP(distill_topk, distill_topk)
CIGN_OP(distill_topk_forward, distill_topk_forward)
CIGN_OP(distill_topk_backward, distill_topk_backward)

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& teacher, const Tensor& index,
                        double temperature, bool tail, bool graph) {
    const at::AutoDispatchBelowADInplaceOrView below;
    if (!graph) return call_distill_topk(x, teacher, index, temperature, tail);
    auto [loss, kept] = call_distill_topk_forward(x, teacher, index, temperature, tail);
    ctx->save_for_backward({x, index, kept});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(6);
    {
      const at::NoGradGuard no_grad;
      out[0] = call_distill_topk_backward(grads[0], saved[0], saved[1], saved[2],
                                          ctx->saved_data["temperature"].toDouble());
    }
    return sealed(std::move(out), "distill_topk_loss");
  }
};

Tensor distill_topk_autograd(const Tensor& x, const Tensor& teacher, const Tensor& index, double temperature,
                             bool tail) {
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK_VALUE(!(grad && teacher.requires_grad()), "teacher_logprobs is a constant of the loss: detach it");
  const bool graph = grad && x.requires_grad();
  if (!graph && !has_tangent(x) && !has_tangent(teacher)) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_distill_topk(x, teacher, index, temperature, tail);
  }
  return Distill::apply(x, teacher, index, temperature, tail, graph);
}

// ---- the operators -------------------------------------------------------------

TORCH_LIBRARY(cign_amd, m) {
  m.def("layernorm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layernorm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  m.def(
      "layernorm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor stats, ScalarType params, bool of_x, "
      "bool of_weight, bool of_bias) -> Tensor[]");
  m.def(
      "class_logprobs(Tensor logits, Tensor? labels, int top_k, float temperature, int ignore_index) -> Tensor[]");
  m.def(
      "class_logprobs_forward(Tensor logits, Tensor? labels, int top_k, float temperature, int ignore_index) "
      "-> Tensor[]");
  m.def(
      "class_logprobs_backward(Tensor? grad_entropy, Tensor? grad_logprob, Tensor logits, Tensor? labels, "
      "Tensor stats, float temperature, int ignore_index) -> Tensor");
  m.def(
      "distill_topk(Tensor logits, Tensor teacher_logprobs, Tensor teacher_index, float temperature, bool tail) "
      "-> Tensor");
  m.def(
      "distill_topk_forward(Tensor logits, Tensor teacher_logprobs, Tensor teacher_index, float temperature, "
      "bool tail) -> (Tensor, Tensor)");
  m.def(
      "distill_topk_backward(Tensor grad, Tensor logits, Tensor teacher_index, Tensor kept, float temperature) "
      "-> Tensor");
}

// On meta tensors the checks run and the results have their shapes.
void kernels(torch::Library& m) {
  m.impl("layernorm", &layernorm);
  m.impl("layernorm_forward", &layernorm_forward);
  m.impl("layernorm_backward", &layernorm_backward);
  m.impl("class_logprobs", &class_logprobs);
  m.impl("class_logprobs_forward", &class_logprobs_forward);
  m.impl("class_logprobs_backward", &class_logprobs_backward);
  m.impl("distill_topk", &distill_topk);
  m.impl("distill_topk_forward", &distill_topk_forward);
  m.impl("distill_topk_backward", &distill_topk_backward);
}

TORCH_LIBRARY_IMPL(cign_amd, CUDA, m) { kernels(m); }

TORCH_LIBRARY_IMPL(cign_amd, Meta, m) { kernels(m); }

TORCH_LIBRARY_IMPL(cign_amd, Autograd, m) {
  m.impl("layernorm", &layernorm_autograd);
  m.impl("class_logprobs", &class_logprobs_autograd);
  m.impl("distill_topk", &distill_topk_autograd);
}

// (logprob, entropy, top_logprobs, top_index), None where not asked for
std::tuple<Optional, Tensor, Optional, Optional> named_logprobs(const Tensor& x, const Optional& labels, int64_t top_k,
                                                                double temperature, int64_t ignore_index) {
  const variable_list r = call_class_logprobs(x, labels, top_k, temperature, ignore_index);
  Optional logprob, top, index;
  if (labels) logprob = r[1];
  if (top_k) {
    top = r[r.size() - 2];
    index = r.back();
  }
  return {logprob, r[0], top, index};
}

}  // namespace

PYBIND11_MODULE(_cign_ops, m) {
  m.doc() = "The operators at the model's output and of a training step, and their autograd nodes.";
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("layernorm", &call_layernorm<Tensor, Optional, Optional, double>, free);
  m.def("class_logprobs", &named_logprobs, free);
  m.def("distill_topk", &call_distill_topk<Tensor, Tensor, Tensor, double, bool>, free);
  cign_ops::bind_step_ops(m);
}
