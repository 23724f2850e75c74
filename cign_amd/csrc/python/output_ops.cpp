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
// The gradients are once differentiable: what a graph of the gradient would
// hold is an error, as once_differentiable makes it.
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <tuple>
#include <utility>

#include "cign_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kStats = 8;  // floats a row that the distillation's backward reads

int32_t code(at::ScalarType t) { return t == at::kFloat ? 0 : 1; }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check(int rc, const char* name) {
  TORCH_CHECK(rc == 0, name, " failed (status ", rc, "): ", cign_last_error());
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// t as [rows, width], values next to each other; a copy only where the leading
// axes do not collapse to one or the last is strided.
Tensor as_rows(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) != 1 && r.size(1) > 1 ? r.contiguous() : r;
}

Tensor like(const Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, t.options().dtype(type));
}

Tensor value(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

Tensor workspace(const Tensor& t, int64_t bytes) { return bytes ? like(t, {bytes}, at::kByte) : Tensor(); }

// A gradient that a graph was asked for: differentiating it raises.
variable_list sealed(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice a function marked with @once_differentiable: ") + name,
      static_cast<int64_t>(defined.size()));
  variable_list out = (*error)(std::move(defined));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// ---- LayerNorm -------------------------------------------------------------

Tensor layernorm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  const int64_t n = rows.size(0), D = rows.size(1);
  const Tensor y = like(x, x.sizes(), x.scalar_type());
  float* mean = nullptr;
  if (stats) {
    *stats = like(x, {2, n}, at::kFloat);
    mean = stats->data_ptr<float>();
  }
  const Tensor& param = weight.defined() ? weight : bias.defined() ? bias : x;
  check(cign_layernorm_fwd(stream_of(x), n, static_cast<int32_t>(D), code(x.scalar_type()), code(param.scalar_type()),
                           rows.data_ptr(), rows.stride(0), ptr(weight), ptr(bias), static_cast<float>(eps),
                           y.data_ptr(), mean, mean ? mean + n : nullptr),
        "cign_layernorm_fwd");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps) {
    Tensor stats;
    Tensor y = layernorm_forward(x, value(weight), value(bias), eps, &stats);
    ctx->save_for_backward({x, value(weight), stats});
    ctx->saved_data["params"] =
        static_cast<int64_t>(weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type());
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
    const c10::DeviceGuard guard(x.device());
    variable_list out(4);
    {
      const at::NoGradGuard no_grad;
      const auto type = static_cast<at::ScalarType>(ctx->saved_data["params"].toInt());
      const Tensor rows = as_rows(x), gy = as_rows(grads[0]);
      const int64_t n = rows.size(0), D = rows.size(1);
      // the edges count the tensors that were given
      if (ctx->needs_input_grad(0)) out[0] = like(x, x.sizes(), x.scalar_type());
      if (weight.defined() && ctx->needs_input_grad(1)) out[1] = like(x, {D}, type);
      if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1))
        out[2] = like(x, {D}, type);
      const bool params = out[1].defined() || out[2].defined();
      const int64_t bytes = params ? cign_layernorm_bwd_workspace_bytes(n, static_cast<int32_t>(D)) : 0;
      const Tensor ws = workspace(x, bytes);
      const float* mean = stats.data_ptr<float>();
      check(cign_layernorm_bwd(stream_of(x), n, static_cast<int32_t>(D), code(x.scalar_type()), code(type),
                               gy.data_ptr(), gy.stride(0), rows.data_ptr(), rows.stride(0), ptr(weight), mean,
                               mean + n, ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(ws), bytes),
            "cign_layernorm_bwd");
    }
    return sealed(std::move(out), "fused_layernorm");
  }
};

Tensor layernorm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  const auto whole = [](const std::optional<Tensor>& t) {
    return t ? std::optional<Tensor>(t->contiguous()) : std::nullopt;
  };
  const std::optional<Tensor> w = whole(weight), b = whole(bias);
  const bool needed = x.requires_grad() || (w && w->requires_grad()) || (b && b->requires_grad());
  if (at::GradMode::is_enabled() && needed) return LayerNorm::apply(x, w, b, eps);
  return layernorm_forward(x, value(w), value(b), eps, nullptr);
}

// ---- log probabilities -------------------------------------------------------

// entropy, then logprob with labels, then top log probabilities and indices with top_k
variable_list logprobs_forward(const Tensor& x, const Tensor& labels, int64_t top_k, double temperature,
                               int64_t ignore_index, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  const int64_t n = rows.size(0);
  const int32_t V = static_cast<int32_t>(rows.size(1)), K = static_cast<int32_t>(top_k), type = code(x.scalar_type());
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  variable_list out{like(x, lead, at::kFloat)};
  Tensor logprob, top, index;
  if (labels.defined()) out.push_back(logprob = like(x, lead, at::kFloat));
  if (top_k) {
    std::vector<int64_t> shape = lead.vec();
    shape.push_back(top_k);
    out.push_back(top = like(x, shape, at::kFloat));
    out.push_back(index = like(x, shape, at::kLong));
  }
  if (stats) *stats = like(x, {n, 4}, at::kFloat);
  const int64_t bytes = cign_class_logprobs_workspace_bytes(type, n, V, K);
  const Tensor ws = workspace(x, bytes);
  check(cign_class_logprobs_fwd(stream_of(x), type, n, V, rows.data_ptr(), rows.stride(0),
                                static_cast<float>(temperature), ptr<int64_t>(labels), ignore_index, K,
                                ptr<float>(logprob), out[0].data_ptr<float>(), ptr<float>(top), ptr<int64_t>(index),
                                stats ? stats->data_ptr<float>() : nullptr, ptr(ws), bytes),
        "cign_class_logprobs_fwd");
  return out;
}

struct Logprobs : torch::autograd::Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& labels,
                               int64_t top_k, double temperature, int64_t ignore_index) {
    Tensor stats;
    variable_list out = logprobs_forward(x, value(labels), top_k, temperature, ignore_index, &stats);
    ctx->save_for_backward({x, value(labels), stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore_index;
    ctx->set_materialize_grads(false);
    if (top_k) ctx->mark_non_differentiable({out[out.size() - 2], out.back()});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &labels = saved[1], &stats = saved[2];
    variable_list out(5);
    const Tensor given = labels.defined() ? grads[1] : Tensor();
    if (!grads[0].defined() && !given.defined()) return out;
    const c10::DeviceGuard guard(x.device());
    {
      const at::NoGradGuard no_grad;
      const Tensor rows = as_rows(x);
      const Tensor ge = grads[0].defined() ? grads[0].contiguous() : Tensor();
      const Tensor gl = given.defined() ? given.contiguous() : Tensor();
      out[0] = like(x, x.sizes(), x.scalar_type());
      check(cign_class_logprobs_bwd(stream_of(x), code(x.scalar_type()), rows.size(0),
                                    static_cast<int32_t>(rows.size(1)), rows.data_ptr(), rows.stride(0),
                                    static_cast<float>(ctx->saved_data["temperature"].toDouble()),
                                    ptr<int64_t>(labels), ctx->saved_data["ignore"].toInt(),
                                    stats.data_ptr<float>(), ptr<float>(gl), ptr<float>(ge), out[0].data_ptr()),
            "cign_class_logprobs_bwd");
    }
    return sealed(std::move(out), "class_logprobs");
  }
};

// (logprob, entropy, top_logprobs, top_index), None where not asked for
std::tuple<std::optional<Tensor>, Tensor, std::optional<Tensor>, std::optional<Tensor>> logprobs(
    const Tensor& x, const std::optional<Tensor>& labels, int64_t top_k, double temperature, int64_t ignore_index) {
  const variable_list r = at::GradMode::is_enabled() && x.requires_grad()
                              ? Logprobs::apply(x, labels, top_k, temperature, ignore_index)
                              : logprobs_forward(x, value(labels), top_k, temperature, ignore_index, nullptr);
  std::optional<Tensor> logprob, top, index;
  if (labels) logprob = r[1];
  if (top_k) {
    top = r[r.size() - 2];
    index = r.back();
  }
  return {logprob, r[0], top, index};
}

// ---- distillation ------------------------------------------------------------

Tensor distill_forward(const Tensor& x, const Tensor& teacher, const Tensor& index, double temperature, bool tail,
                       Tensor* kept) {
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  const int64_t n = rows.size(0), K = index.size(-1);
  const int32_t V = static_cast<int32_t>(rows.size(1)), type = code(x.scalar_type());
  Tensor loss = like(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  float* stats = nullptr;
  if (kept) {  // the rows' statistics, then their lists' masses
    *kept = like(x, {n * (kStats + K)}, at::kFloat);
    stats = kept->data_ptr<float>();
  }
  const int64_t bytes = cign_distill_topk_workspace_bytes(type, n, V);
  const Tensor ws = workspace(x, bytes);
  check(cign_distill_topk_fwd(stream_of(x), type, n, V, rows.data_ptr(), rows.stride(0),
                              static_cast<float>(temperature), tail, static_cast<int32_t>(K),
                              teacher.data_ptr<float>(), index.data_ptr<int64_t>(), loss.data_ptr<float>(), stats,
                              stats ? stats + n * kStats : nullptr, ptr(ws), bytes),
        "cign_distill_topk_fwd");
  return loss;
}

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& teacher, const Tensor& index,
                        double temperature, bool tail) {
    Tensor kept;
    Tensor loss = distill_forward(x, teacher, index, temperature, tail, &kept);
    ctx->save_for_backward({x, index, kept});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &index = saved[1], &kept = saved[2];
    const c10::DeviceGuard guard(x.device());
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      const Tensor rows = as_rows(x), g = grads[0].contiguous();
      const int64_t n = rows.size(0);
      out[0] = like(x, x.sizes(), x.scalar_type());
      const float* stats = kept.data_ptr<float>();
      check(cign_distill_topk_bwd(stream_of(x), code(x.scalar_type()), n, static_cast<int32_t>(rows.size(1)),
                                  rows.data_ptr(), rows.stride(0),
                                  static_cast<float>(ctx->saved_data["temperature"].toDouble()),
                                  static_cast<int32_t>(index.size(-1)), index.data_ptr<int64_t>(), stats,
                                  stats + n * kStats, g.data_ptr<float>(), out[0].data_ptr()),
            "cign_distill_topk_bwd");
    }
    return sealed(std::move(out), "distill_topk_loss");
  }
};

Tensor distill_topk(const Tensor& x, const Tensor& teacher, const Tensor& index, double temperature, bool tail) {
  if (at::GradMode::is_enabled() && x.requires_grad()) return Distill::apply(x, teacher, index, temperature, tail);
  return distill_forward(x, teacher, index, temperature, tail, nullptr);
}

}  // namespace

PYBIND11_MODULE(_cign_ops, m) {
  m.doc() = "Autograd nodes of the operators at the model's output.";
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("layernorm", &layernorm, free);
  m.def("class_logprobs", &logprobs, free);
  m.def("distill_topk", &distill_topk, free);
}
