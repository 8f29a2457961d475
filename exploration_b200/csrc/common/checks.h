// Argument checks of the decoding operators, raised as Python ValueErrors.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>

namespace eb {

// A gradient would have to flow through `t`: backward, or forward as a dual number's tangent.
inline bool wants_grad(const at::Tensor& t) {
  return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(/*level=*/0).defined();
}

template <typename... Rest>
bool same_device(const at::Tensor& first, const Rest&... rest) {
  return ((rest.device() == first.device()) && ...);
}

inline bool native_dtype(const at::Tensor& t) {
  const auto type = t.scalar_type();
  return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

}  // namespace eb
