// The operators of a training step as operators of torch's dispatcher: the
// boundary of two blocks, the cross entropy of a linear classifier, the global
// norm of gradients. Checks, derivatives and traces as those of output_ops.cpp.
#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <array>

#include "ops.h"

namespace {

using namespace cign_ops;

// ---- block boundary ----------------------------------------------------------

enum Gate : int32_t { kNoGate = 0, kRowGate = 1, kValueGate = 2 };

struct Boundary {
  int64_t n, D;
  Tensor branch, residual, gate, vec[5];  // rows; vectors whole
  at::ScalarType params;
  int32_t kind;
};

Boundary check_boundary(const Tensor& branch, const Tensor& residual, const Optional& gate,
                        const std::array<Optional, 5>& vec) {
  static const char* const names[5] = {"post_weight", "post_bias", "scale", "next_weight", "next_bias"};
  check_rows(branch, "branch");
  check_beside(residual, branch, "residual", branch.scalar_type(), branch.sizes());
  Boundary b;
  b.D = branch.size(-1);
  b.n = row_count(branch);
  b.kind = kNoGate;
  if (gate) {
    std::vector<int64_t> one = lead(branch).vec();
    one.push_back(1);
    b.kind = gate->dim() == branch.dim() && gate->sizes() == at::IntArrayRef(one) ? kRowGate : kValueGate;
    check_beside(*gate, branch, "gate", branch.scalar_type(), b.kind == kRowGate ? at::IntArrayRef(one) : branch.sizes());
  }
  b.params = branch.scalar_type();
  for (int i = 4; i >= 0; --i)
    if (vec[i]) b.params = vec[i]->scalar_type();
  for (int i = 0; i < 5; ++i)
    if (vec[i]) {
      TORCH_CHECK_TYPE(vec[i]->scalar_type() == b.params && (b.params == at::kFloat || b.params == branch.scalar_type()),
                       "the vectors must all be float32 or all of branch's type");
      check_beside(*vec[i], branch, names[i], b.params, {b.D});
      b.vec[i] = vec[i]->contiguous();
    }
  if (branch.is_meta()) return b;
  b.branch = as_rows(branch);
  b.residual = as_rows(residual);
  if (gate) b.gate = as_rows(*gate);
  return b;
}

int64_t gate_stride(const Boundary& b) { return b.gate.defined() ? b.gate.stride(0) : 0; }

std::tuple<Tensor, Tensor> run_boundary(const Tensor& branch, const Tensor& residual, const Optional& w1,
                                        const Optional& b1, const Optional& scale, const Optional& gate,
                                        const Optional& w2, const Optional& b2, double eps, bool layer, Tensor* stats) {
  const c10::OptionalDeviceGuard guard(branch.is_cuda() ? std::optional<c10::Device>(branch.device()) : std::nullopt);
  const Boundary b = check_boundary(branch, residual, gate, {w1, b1, scale, w2, b2});
  Tensor hidden = like(branch, branch.sizes(), branch.scalar_type());
  Tensor y = like(branch, branch.sizes(), branch.scalar_type());
  if (stats) *stats = like(branch, {4, b.n}, at::kFloat);
  if (branch.is_meta()) return {hidden, y};
  check(cign_block_boundary_fwd(stream_of(branch), b.n, static_cast<int32_t>(b.D), code(branch.scalar_type()),
                                code(b.params), layer, b.kind, b.branch.data_ptr(), b.branch.stride(0),
                                b.residual.data_ptr(), b.residual.stride(0), ptr(b.gate), gate_stride(b), ptr(b.vec[0]),
                                ptr(b.vec[1]), ptr(b.vec[2]), ptr(b.vec[3]), ptr(b.vec[4]), static_cast<float>(eps),
                                hidden.data_ptr(), y.data_ptr(), stats ? stats->data_ptr<float>() : nullptr),
        "cign_block_boundary_fwd");
  return {hidden, y};
}

std::tuple<Tensor, Tensor> block_boundary(const Tensor& branch, const Tensor& residual, const Optional& w1,
                                          const Optional& b1, const Optional& scale, const Optional& gate,
                                          const Optional& w2, const Optional& b2, double eps, bool layer) {
  return run_boundary(branch, residual, w1, b1, scale, gate, w2, b2, eps, layer, nullptr);
}

// hidden, y and the rows' statistics
std::tuple<Tensor, Tensor, Tensor> block_boundary_forward(const Tensor& branch, const Tensor& residual,
                                                          const Optional& w1, const Optional& b1, const Optional& scale,
                                                          const Optional& gate, const Optional& w2, const Optional& b2,
                                                          double eps, bool layer) {
  Tensor stats;
  auto [hidden, y] = run_boundary(branch, residual, w1, b1, scale, gate, w2, b2, eps, layer, &stats);
  return {hidden, y, stats};
}

// The gradients asked for by the bits of `of`: branch, residual, gate, post_weight,
// post_bias, scale, next_weight, next_bias. next_bias's own value is not read.
variable_list block_boundary_backward(const Optional& g1, const Optional& g2, const Tensor& branch,
                                      const Tensor& residual, const Optional& w1, const Optional& b1,
                                      const Optional& scale, const Optional& gate, const Optional& w2,
                                      const Tensor& stats, at::ScalarType params, bool layer, int64_t of) {
  const c10::OptionalDeviceGuard guard(branch.is_cuda() ? std::optional<c10::Device>(branch.device()) : std::nullopt);
  const Boundary b = check_boundary(branch, residual, gate, {w1, b1, scale, w2, std::nullopt});
  TORCH_CHECK_TYPE(params == at::kFloat || params == branch.scalar_type(),
                   "the vectors are float32 or of branch's type");
  for (const Optional& v : {w1, b1, scale, w2})
    TORCH_CHECK_TYPE(!v || v->scalar_type() == params, "the vectors must all be of one type");
  check_beside(stats, branch, "the statistics", at::kFloat, {4, b.n});
  for (const Optional& g : {g1, g2})
    if (g) check_beside(*g, branch, "the gradient", branch.scalar_type(), branch.sizes());
  Tensor grads[8];
  variable_list out;
  for (int i = 0; i < 8; ++i) {
    if (!((of >> i) & 1)) continue;
    if (i == 2) {
      TORCH_CHECK_VALUE(gate.has_value(), "no gate to take the gradient of");
      grads[i] = like(branch, gate->sizes(), branch.scalar_type());
    } else {
      grads[i] = i < 2 ? like(branch, branch.sizes(), branch.scalar_type()) : like(branch, {b.D}, params);
    }
    out.push_back(grads[i]);
  }
  if (branch.is_meta()) return out;
  const Tensor r1 = g1 ? as_rows(*g1) : Tensor(), r2 = g2 ? as_rows(*g2) : Tensor(), kept = stats.contiguous();
  const int64_t bytes = of >> 3 ? cign_block_boundary_bwd_workspace_bytes(b.n, static_cast<int32_t>(b.D)) : 0;
  const Tensor ws = workspace(branch, bytes);
  check(cign_block_boundary_bwd(
            stream_of(branch), b.n, static_cast<int32_t>(b.D), code(branch.scalar_type()), code(params), layer, b.kind,
            ptr(r1), r1.defined() ? r1.stride(0) : 0, ptr(r2), r2.defined() ? r2.stride(0) : 0, b.branch.data_ptr(),
            b.branch.stride(0), b.residual.data_ptr(), b.residual.stride(0), ptr(b.gate), gate_stride(b), ptr(b.vec[0]),
            ptr(b.vec[1]), ptr(b.vec[2]), ptr(b.vec[3]), kept.data_ptr<float>(), ptr(grads[0]), ptr(grads[1]),
            ptr(grads[2]), ptr(grads[3]), ptr(grads[4]), ptr(grads[5]), ptr(grads[6]), ptr(grads[7]), ptr(ws), bytes),
        "cign_block_boundary_bwd");
  return out;
}

CIGN_OP(block_boundary, block_boundary)
CIGN_OP(block_boundary_forward, block_boundary_forward)
CIGN_OP(block_boundary_backward, block_boundary_backward)

struct BlockBoundary : torch::autograd::Function<BlockBoundary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& branch, const Tensor& residual, const Optional& w1,
                               const Optional& b1, const Optional& scale, const Optional& gate, const Optional& w2,
                               const Optional& b2, double eps, bool layer, bool graph) {
    const at::AutoDispatchBelowADInplaceOrView below;
    if (!graph) {
      auto [hidden, y] = call_block_boundary(branch, residual, w1, b1, scale, gate, w2, b2, eps, layer);
      return {hidden, y};
    }
    auto [hidden, y, stats] = call_block_boundary_forward(branch, residual, w1, b1, scale, gate, w2, b2, eps, layer);
    ctx->save_for_backward({branch, residual, value(w1), value(b1), value(scale), value(gate), value(w2), stats});
    int64_t given = 0;
    const Optional* const all[8] = {nullptr, nullptr, &w1, &b1, &scale, &gate, &w2, &b2};
    at::ScalarType params = branch.scalar_type();
    for (int i = 2; i < 8; ++i)
      if (*all[i]) {
        given |= 1 << i;
        if (i != 5) params = (*all[i])->scalar_type();
      }
    ctx->saved_data["given"] = given | 3;
    ctx->saved_data["params"] = static_cast<int64_t>(params);
    ctx->saved_data["layer"] = layer;
    ctx->set_materialize_grads(false);
    return {hidden, y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(11);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    // places of the inputs (branch, residual, w1, b1, scale, gate, w2, b2) among the
    // gradients' bits; the graph's edges count the tensors that were given
    static constexpr int bit[8] = {0, 1, 3, 4, 5, 2, 6, 7};
    const int64_t given = ctx->saved_data["given"].toInt();
    int64_t of = 0;
    int place[8];
    for (int i = 0, edge = 0; i < 8; ++i) {
      if (!((given >> i) & 1)) continue;
      if (ctx->needs_input_grad(edge++)) of |= 1 << bit[i];
    }
    for (int i = 0; i < 8; ++i) place[bit[i]] = i;
    {
      const at::NoGradGuard no_grad;
      const at::AutoDispatchBelowADInplaceOrView below;
      const variable_list got = call_block_boundary_backward(
          optional(grads[0]), optional(grads[1]), saved[0], saved[1], optional(saved[2]), optional(saved[3]),
          optional(saved[4]), optional(saved[5]), optional(saved[6]), saved[7],
          static_cast<at::ScalarType>(ctx->saved_data["params"].toInt()), ctx->saved_data["layer"].toBool(), of);
      for (int i = 0, k = 0; i < 8; ++i)
        if ((of >> i) & 1) out[place[i]] = got[k++];
    }
    return sealed(std::move(out), "fused_gated_residual_norm");
  }
};

bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const Optional& t) { return t && t->requires_grad(); }

std::tuple<Tensor, Tensor> block_boundary_autograd(const Tensor& branch, const Tensor& residual, const Optional& w1,
                                                   const Optional& b1, const Optional& scale, const Optional& gate,
                                                   const Optional& w2, const Optional& b2, double eps, bool layer) {
  const bool graph = at::GradMode::is_enabled() && (wants(branch) || wants(residual) || wants(w1) || wants(b1) ||
                                                    wants(scale) || wants(gate) || wants(w2) || wants(b2));
  if (!graph && !has_tangent(branch) && !has_tangent(residual) && !has_tangent(w1) && !has_tangent(b1) &&
      !has_tangent(scale) && !has_tangent(gate) && !has_tangent(w2) && !has_tangent(b2)) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_block_boundary(branch, residual, w1, b1, scale, gate, w2, b2, eps, layer);
  }
  const variable_list r =
      BlockBoundary::apply(branch, residual, w1, b1, scale, gate, w2, b2, eps, layer, graph);
  return {r[0], r[1]};
}

// ---- cross entropy of a linear classifier ------------------------------------

struct Classifier {
  int64_t n, D, V;
  Tensor x, weight, bias, labels;
  int32_t type, bias_type;
};

Classifier check_classifier(const Tensor& x, const Tensor& weight, const Tensor& labels, const Optional& bias) {
  check_rows(x, "x");
  Classifier c;
  c.D = x.size(-1);
  c.n = row_count(x);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) == c.D, "weight must be [V, ", c.D,
                    "], got ", weight.sizes());
  c.V = weight.size(0);
  check_beside(weight, x, "weight", x.scalar_type(), {c.V, c.D});
  check_beside(labels, x, "labels", at::kLong, lead(x));
  c.type = code(x.scalar_type());
  c.bias_type = c.type;
  if (bias) {
    TORCH_CHECK_TYPE(bias->scalar_type() == at::kFloat || bias->scalar_type() == x.scalar_type(),
                     "bias must be float32 or of x's type");
    check_beside(*bias, x, "bias", bias->scalar_type(), {c.V});
    c.bias = bias->contiguous();
    c.bias_type = code(bias->scalar_type());
  }
  TORCH_CHECK_VALUE(c.V <= std::numeric_limits<int32_t>::max(), "too many classes");
  if (x.is_meta()) return c;
  c.x = as_rows(x);
  c.weight = as_rows(weight);
  c.labels = labels.contiguous();
  return c;
}

int64_t xent_bytes(const Classifier& c, int32_t of) {
  return cign_linear_xent_workspace_bytes(c.type, c.n, static_cast<int32_t>(c.V), static_cast<int32_t>(c.D),
                                          c.x.data_ptr(), c.x.stride(0), c.weight.data_ptr(), c.weight.stride(0), of);
}

// loss and logsumexp
std::tuple<Tensor, Tensor> linear_xent(const Tensor& x, const Tensor& weight, const Tensor& labels,
                                       const Optional& bias, int64_t ignore_index) {
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::optional<c10::Device>(x.device()) : std::nullopt);
  const Classifier c = check_classifier(x, weight, labels, bias);
  Tensor loss = like(x, lead(x), at::kFloat), lse = like(x, lead(x), at::kFloat);
  if (x.is_meta()) return {loss, lse};
  const int64_t bytes = xent_bytes(c, 0);
  const Tensor ws = workspace(x, bytes);
  check(cign_linear_xent_fwd(stream_of(x), c.type, c.n, static_cast<int32_t>(c.V), static_cast<int32_t>(c.D),
                             c.x.data_ptr(), c.x.stride(0), c.weight.data_ptr(), c.weight.stride(0), ptr(c.bias),
                             c.bias_type, c.labels.data_ptr<int64_t>(), ignore_index, loss.data_ptr<float>(),
                             lse.data_ptr<float>(), ptr(ws), bytes),
        "cign_linear_xent_fwd");
  return {loss, lse};
}

// the gradients asked for of (x, weight, bias)
variable_list linear_xent_backward(const Optional& grad_loss, const Optional& grad_lse, const Tensor& x,
                                   const Tensor& weight, const Tensor& labels, const Optional& bias, const Tensor& lse_,
                                   int64_t ignore_index, bool of_x, bool of_weight, bool of_bias) {
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::optional<c10::Device>(x.device()) : std::nullopt);
  const Classifier c = check_classifier(x, weight, labels, bias);
  check_beside(lse_, x, "logsumexp", at::kFloat, lead(x));
  if (grad_loss) check_beside(*grad_loss, x, "the loss's gradient", at::kFloat, lead(x));
  if (grad_lse) check_beside(*grad_lse, x, "logsumexp's gradient", at::kFloat, lead(x));
  TORCH_CHECK_VALUE(grad_loss || grad_lse, "no gradient given");
  TORCH_CHECK_VALUE(!of_bias || bias, "no bias to take the gradient of");
  Tensor gx, gw, gb;
  variable_list out;
  if (of_x) out.push_back(gx = like(x, x.sizes(), x.scalar_type()));
  if (of_weight) out.push_back(gw = like(x, weight.sizes(), x.scalar_type()));
  if (of_bias) out.push_back(gb = like(x, {c.V}, bias->scalar_type()));
  if (x.is_meta()) return out;
  if (c.n == 0) {
    for (Tensor& t : out) t.zero_();
    return out;
  }
  const Tensor g1 = whole(grad_loss), g2 = whole(grad_lse), lse = lse_.contiguous();
  const int32_t of = (of_x ? 1 : 0) | (of_weight ? 2 : 0) | (of_bias ? 4 : 0);
  const int64_t bytes = of ? xent_bytes(c, of) : 0;
  const Tensor ws = workspace(x, bytes);
  check(cign_linear_xent_bwd(stream_of(x), c.type, c.n, static_cast<int32_t>(c.V), static_cast<int32_t>(c.D),
                             c.x.data_ptr(), c.x.stride(0), c.weight.data_ptr(), c.weight.stride(0), ptr(c.bias),
                             c.bias_type, c.labels.data_ptr<int64_t>(), ignore_index, lse.data_ptr<float>(),
                             ptr<float>(g1), ptr<float>(g2), ptr(gx), ptr(gw), ptr(gb), ptr(ws), bytes),
        "cign_linear_xent_bwd");
  return out;
}

CIGN_OP(linear_xent, linear_xent)
CIGN_OP(linear_xent_backward, linear_xent_backward)

struct LinearXent : torch::autograd::Function<LinearXent> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& labels,
                               const Optional& bias, int64_t ignore_index, bool graph) {
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, lse] = call_linear_xent(x, weight, labels, bias, ignore_index);
    if (graph) {
      ctx->save_for_backward({x, weight, labels, value(bias), lse});
      ctx->saved_data["ignore"] = ignore_index;
      ctx->set_materialize_grads(false);
    }
    return {loss, lse};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(6);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const at::AutoDispatchBelowADInplaceOrView below;
      const bool of[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                          saved[3].defined() && ctx->needs_input_grad(3)};
      const variable_list got =
          call_linear_xent_backward(optional(grads[0]), optional(grads[1]), saved[0], saved[1], saved[2],
                                    optional(saved[3]), saved[4], ctx->saved_data["ignore"].toInt(), of[0], of[1], of[2]);
      static constexpr int place[3] = {0, 1, 3};
      for (size_t i = 0, k = 0; i < 3; ++i)
        if (of[i]) out[place[i]] = got[k++];
    }
    return sealed(std::move(out), "linear_cross_entropy");
  }
};

std::tuple<Tensor, Tensor> linear_xent_autograd(const Tensor& x, const Tensor& weight, const Tensor& labels,
                                                const Optional& bias, int64_t ignore_index) {
  const bool graph = at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias));
  if (!graph && !has_tangent(x) && !has_tangent(weight) && !has_tangent(bias)) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_linear_xent(x, weight, labels, bias, ignore_index);
  }
  const variable_list r = LinearXent::apply(x, weight, labels, bias, ignore_index, graph);
  return {r[0], r[1]};
}

// ---- global norm of gradients --------------------------------------------------

void check_grads(at::TensorList grads, const char* name) {
  for (const Tensor& g : grads) {
    TORCH_CHECK_TYPE((g.is_cuda() || g.is_meta()) && g.layout() == at::kStrided &&
                         (g.scalar_type() == at::kFloat || g.scalar_type() == at::kBFloat16),
                     name, " must be CUDA float32 or bfloat16");
    TORCH_CHECK_VALUE(g.device() == grads[0].device(), name, " must be on one device, got ", grads[0].device(), " and ",
                      g.device());
  }
}

// A run of memory for each tensor: itself where its values fill one, else a copy.
struct Flat {
  std::vector<Tensor> held;
  std::vector<const void*> at;
  std::vector<int64_t> sizes;
  std::vector<int32_t> types;
  void add(const Tensor& t) {
    held.push_back(t);
    at.push_back(t.numel() ? t.data_ptr() : nullptr);
    sizes.push_back(t.numel());
    types.push_back(code(t.scalar_type()));
  }
  int32_t count() const { return static_cast<int32_t>(held.size()); }
};

bool fills(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

Tensor global_grad_norm(at::TensorList grads) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  check_grads(grads, "gradients");
  const Tensor& first = grads[0];
  Tensor norm = like(first, {}, at::kFloat);
  if (first.is_meta()) return norm;
  const c10::DeviceGuard guard(first.device());
  Flat flat;
  for (const Tensor& g : grads) flat.add(fills(g) ? g : g.contiguous());
  const int64_t bytes = cign_grad_norm_workspace_bytes(flat.count(), flat.sizes.data());
  const Tensor ws = workspace(first, bytes);
  check(cign_grad_norm(stream_of(first), flat.count(), flat.at.data(), flat.sizes.data(), flat.types.data(),
                       norm.data_ptr<float>(), ptr(ws), bytes),
        "cign_grad_norm");
  return norm;
}

// The bytes between a tensor's first and last value, and whose they are.
struct Span {
  uintptr_t from, to;
  size_t index;
  bool out;
};

Span span_of(const Tensor& t, size_t index, bool out) {
  uintptr_t from = reinterpret_cast<uintptr_t>(t.data_ptr());
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {from, from + static_cast<uintptr_t>((last + 1) * t.element_size()), index, out};
}

bool same_place(const Tensor& a, const Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.scalar_type() == b.scalar_type() && a.strides() == b.strides();
}

// Every written tensor apart from the others, and from all gradients but its own
// (whose place it may be).
void check_apart(at::TensorList grads, at::TensorList out) {
  std::vector<Span> spans;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (grads[i].numel() == 0) continue;
    TORCH_CHECK_VALUE(at::has_internal_overlap(out[i]) != at::MemOverlap::Yes,
                      "a gradient that is written must have a place for each value");
    spans.push_back(span_of(out[i], i, true));
    if (!same_place(grads[i], out[i])) spans.push_back(span_of(grads[i], i, false));
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  // the furthest ends of what came before, of any span and of written ones
  uintptr_t any = 0, written = 0;
  for (const Span& s : spans) {
    TORCH_CHECK_VALUE(s.from >= (s.out ? any : written),
                      "gradients that are written must not share memory with each other or with other gradients");
    any = std::max(any, s.to);
    if (s.out) written = std::max(written, s.to);
  }
}

Tensor clip_grad_norm(at::TensorList grads, double max_norm, at::TensorList out) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must not be negative, got ", max_norm);
  TORCH_CHECK_VALUE(out.size() == grads.size(), "out must have ", grads.size(), " tensors, got ", out.size());
  check_grads(grads, "gradients");
  for (size_t i = 0; i < grads.size(); ++i) check_beside(out[i], grads[i], "out", grads[i].scalar_type(), grads[i].sizes());
  const Tensor& first = grads[0];
  Tensor norm = like(first, {}, at::kFloat);
  if (first.is_meta()) return norm;
  check_apart(grads, out);
  const c10::DeviceGuard guard(first.device());
  Flat from, to;
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& g = grads[i];
    const Tensor& o = out[i];
    if (fills(g) && fills(o) && g.strides() == o.strides()) {
      from.add(g);
      to.add(o);
    } else {
      from.add(g.contiguous());
      to.add(o.is_contiguous() ? o : like(o, o.sizes(), o.scalar_type()));
    }
  }
  std::vector<void*> at;
  for (const Tensor& t : to.held) at.push_back(t.numel() ? t.data_ptr() : nullptr);
  const int64_t bytes = cign_grad_norm_workspace_bytes(from.count(), from.sizes.data());
  const Tensor ws = workspace(first, bytes);
  check(cign_clip_grad_norm(stream_of(first), from.count(), from.at.data(), from.sizes.data(), from.types.data(),
                            static_cast<float>(max_norm), at.data(), norm.data_ptr<float>(), ptr(ws), bytes),
        "cign_clip_grad_norm");
  for (size_t i = 0; i < grads.size(); ++i)
    if (!to.held[i].is_same(out[i])) const_cast<Tensor&>(out[i]).copy_(to.held[i]);
  return norm;
}

CIGN_OP(global_grad_norm, global_grad_norm)
CIGN_OP(clip_grad_norm, clip_grad_norm)

Tensor global_grad_norm_autograd(at::TensorList grads) {
  const at::AutoDispatchBelowADInplaceOrView below;
  return call_global_grad_norm(grads);
}

Tensor clip_grad_norm_autograd(at::TensorList grads, double max_norm, at::TensorList out) {
  for (const Tensor& t : out)
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()),
                "a gradient that requires grad is clipped under torch.no_grad()");
  Tensor norm;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    norm = call_clip_grad_norm(grads, max_norm, out);
  }
  for (const Tensor& t : out)
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
  return norm;
}

// ---- the operators ---------------------------------------------------------------

TORCH_LIBRARY_FRAGMENT(cign_amd, m) {
  m.def(
      "block_boundary(Tensor branch, Tensor residual, Tensor? post_weight, Tensor? post_bias, Tensor? scale, "
      "Tensor? gate, Tensor? next_weight, Tensor? next_bias, float eps, bool layer) -> (Tensor, Tensor)");
  m.def(
      "block_boundary_forward(Tensor branch, Tensor residual, Tensor? post_weight, Tensor? post_bias, Tensor? scale, "
      "Tensor? gate, Tensor? next_weight, Tensor? next_bias, float eps, bool layer) -> (Tensor, Tensor, Tensor)");
  m.def(
      "block_boundary_backward(Tensor? grad_hidden, Tensor? grad_y, Tensor branch, Tensor residual, "
      "Tensor? post_weight, Tensor? post_bias, Tensor? scale, Tensor? gate, Tensor? next_weight, Tensor stats, "
      "ScalarType params, bool layer, int of) -> Tensor[]");
  m.def("linear_xent(Tensor x, Tensor weight, Tensor labels, Tensor? bias, int ignore_index) -> (Tensor, Tensor)");
  m.def(
      "linear_xent_backward(Tensor? grad_loss, Tensor? grad_logsumexp, Tensor x, Tensor weight, Tensor labels, "
      "Tensor? bias, Tensor logsumexp, int ignore_index, bool of_x, bool of_weight, bool of_bias) -> Tensor[]");
  m.def("global_grad_norm(Tensor[] grads) -> Tensor");
  m.def("clip_grad_norm(Tensor[] grads, float max_norm, Tensor(a!)[] out) -> Tensor");
}

void kernels(torch::Library& m) {
  m.impl("block_boundary", &block_boundary);
  m.impl("block_boundary_forward", &block_boundary_forward);
  m.impl("block_boundary_backward", &block_boundary_backward);
  m.impl("linear_xent", &linear_xent);
  m.impl("linear_xent_backward", &linear_xent_backward);
  m.impl("global_grad_norm", &global_grad_norm);
  m.impl("clip_grad_norm", &clip_grad_norm);
}

TORCH_LIBRARY_IMPL(cign_amd, CUDA, m) { kernels(m); }

TORCH_LIBRARY_IMPL(cign_amd, Meta, m) { kernels(m); }

TORCH_LIBRARY_IMPL(cign_amd, Autograd, m) {
  m.impl("block_boundary", &block_boundary_autograd);
  m.impl("linear_xent", &linear_xent_autograd);
  m.impl("global_grad_norm", &global_grad_norm_autograd);
  m.impl("clip_grad_norm", &clip_grad_norm_autograd);
}

Tensor bound_global_grad_norm(const std::vector<Tensor>& grads) { return call_global_grad_norm(at::TensorList(grads)); }

// in place without `out`
Tensor bound_clip_grad_norm(const std::vector<Tensor>& grads, double max_norm,
                            const std::optional<std::vector<Tensor>>& out) {
  return call_clip_grad_norm(at::TensorList(grads), max_norm, at::TensorList(out ? *out : grads));
}

}  // namespace

void cign_ops::bind_step_ops(pybind11::module_& m) {
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("block_boundary",
        &call_block_boundary<Tensor, Tensor, Optional, Optional, Optional, Optional, Optional, Optional, double, bool>,
        free);
  m.def("linear_xent", &call_linear_xent<Tensor, Tensor, Tensor, Optional, int64_t>, free);
  m.def("global_grad_norm", &bound_global_grad_norm, free);
  m.def("clip_grad_norm", &bound_clip_grad_norm, free);
}
