// Checks shared by paged_append and paged_attention (the Python module makes the
// same ones for CPU tensors, with the same messages).
#pragma once

#include "../common/checks.h"

namespace eb {
namespace paged {

inline void check_cache(const at::Tensor& x, const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& tables, const at::Tensor& positions) {
  TORCH_CHECK_VALUE(x.dim() == 4 && k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() &&
                        x.size(3) == k_cache.size(3),
                    "expected rows [batch, tokens, heads, head_dim] and caches [pages, kv_heads, page, head_dim]");
  const int64_t page = k_cache.size(2), dim = k_cache.size(3);
  TORCH_CHECK_VALUE(page >= 16 && (page & (page - 1)) == 0, "page must be a power of two of at least 16");
  TORCH_CHECK_VALUE(dim % 2 == 0 && dim >= 2 && dim <= 256, "head_dim must be even and at most 256");
  TORCH_CHECK_VALUE(k_cache.size(1) >= 1 && x.size(2) >= 1 && x.size(2) % k_cache.size(1) == 0,
                    "query heads must be a positive multiple of the cache's heads");
  TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(0) == x.size(0) && positions.size(1) == x.size(1) &&
                        tables.dim() == 2 && tables.size(0) == x.size(0),
                    "expected positions [batch, tokens] and tables [batch, width]");
  TORCH_CHECK_VALUE((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
                        tables.scalar_type() == at::kInt,
                    "positions must be int32 or int64 and tables int32");
  TORCH_CHECK_VALUE(x.scalar_type() == k_cache.scalar_type() && x.scalar_type() == v_cache.scalar_type(),
                    "rows and caches must have one dtype");
  TORCH_CHECK_VALUE(same_device(x, k_cache, v_cache, tables, positions), "all tensors must be on one device");
  TORCH_CHECK_VALUE(!wants_grad(x) && !wants_grad(k_cache) && !wants_grad(v_cache),
                    "paged operators are for inference: they have no gradient");
  TORCH_CHECK_VALUE(native_dtype(x), "the native paged operators take fp32, fp16 or bf16");
  TORCH_CHECK_VALUE(k_cache.is_contiguous() && v_cache.is_contiguous(), "cache pools must be contiguous");
}

inline at::Tensor int32(const at::Tensor& t) { return t.to(at::kInt).contiguous(); }

}  // namespace paged
}  // namespace eb
