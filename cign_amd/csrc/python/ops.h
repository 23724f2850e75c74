// What the torch operators of _cign_ops.so share: checks, allocations, the current
// stream, and what makes a gradient once differentiable. Host code only.
#pragma once

#include <ATen/core/Tensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <limits>
#include <optional>
#include <tuple>
#include <utility>

#include "cign_amd.h"

namespace cign_ops {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

inline int32_t code(at::ScalarType t) { return t == at::kFloat ? 0 : 1; }

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

inline void check(int rc, const char* name) {
  TORCH_CHECK(rc == 0, name, " failed (status ", rc, "): ", cign_last_error());
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// t as [rows, width], values next to each other; a copy only where the leading
// axes do not collapse to one or the last is strided.
inline Tensor as_rows(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) != 1 && r.size(1) > 1 ? r.contiguous() : r;
}

inline Tensor like(const Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, t.options().dtype(type));
}

inline Tensor value(const Optional& t) { return t ? *t : Tensor(); }

inline Tensor whole(const Optional& t) { return t ? t->contiguous() : Tensor(); }

inline Optional optional(const Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }

inline Tensor workspace(const Tensor& t, int64_t bytes) { return bytes ? like(t, {bytes}, at::kByte) : Tensor(); }

inline at::IntArrayRef lead(const Tensor& x) { return x.sizes().slice(0, x.dim() - 1); }

inline int64_t row_count(const Tensor& x) { return x.numel() / x.size(-1); }

inline void check_rows(const Tensor& x, const char* name) {
  TORCH_CHECK_TYPE((x.is_cuda() || x.is_meta()) && x.layout() == at::kStrided &&
                       (x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16),
                   name, " must be CUDA float32 or bfloat16");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= std::numeric_limits<int32_t>::max(), name,
                    " must be [..., D], got ", x.sizes());
}

// t beside x: of this type and shape, on its device
inline void check_beside(const Tensor& t, const Tensor& x, const char* name, at::ScalarType type, at::IntArrayRef shape) {
  TORCH_CHECK_TYPE(t.scalar_type() == type && t.layout() == at::kStrided, name, " must be ", type);
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
}

inline bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }

inline bool has_tangent(const Optional& t) { return t && has_tangent(*t); }

// A gradient that a graph was asked for: differentiating it raises.
inline variable_list sealed(variable_list grads, const char* name) {
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

template <typename F>
c10::TypedOperatorHandle<F> handle(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
// The operator cign_amd::NAME, whose kernel is KERNEL.
#define CIGN_OP(NAME, KERNEL)                                               \
  template <typename... Args>                                               \
  decltype(auto) call_##NAME(const Args&... args) {                         \
    static const auto op = handle("cign_amd::" #NAME, &KERNEL);             \
    return op.call(args...);                                                \
  }

// step_ops.cpp
void bind_step_ops(pybind11::module_& m);

}  // namespace cign_ops
