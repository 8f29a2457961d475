// Argument checks of the decoding operators, raised as Python ValueErrors.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>

namespace eb {

inline bool wants_grad(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

template <typename... Rest>
bool same_device(const at::Tensor& first, const Rest&... rest) {
  return ((rest.device() == first.device()) && ...);
}

inline bool native_dtype(const at::Tensor& t) {
  const auto type = t.scalar_type();
  return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

}  // namespace eb
