// Entry point of paged_attention: argument block and choice of kernel.
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>

#include "paged_launch.h"

namespace eb {

using paged::Args;

namespace {

// Few rows of a key head: the kernel bound by the read of the cache.
bool rows_path(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache) {
  const int64_t dim = q.size(3);
  auto aligned = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; };
  return q.scalar_type() != at::kFloat && (dim == 64 || dim == 128) && aligned(q) && aligned(k_cache) &&
         aligned(v_cache);
}

}  // namespace

std::string paged_attention_path(const at::Tensor& q, const at::Tensor& k_cache) {
  return rows_path(q, k_cache, k_cache) ? "rows" : "cuda_core";
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& tables, const at::Tensor& positions) {
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = at::empty_like(q);
  if (q.numel() == 0) return out;
  TORCH_CHECK(q.size(0) * q.size(1) * q.size(2) < (1LL << 31), "paged_attention: too many rows");
  TORCH_CHECK(tables.size(1) * k_cache.size(2) < (1LL << 30), "paged_attention: tables are too wide");
  if (tables.size(1) == 0 || k_cache.size(0) == 0) return out.zero_();
  Args args{};
  args.q = q.data_ptr();
  args.k = k_cache.data_ptr();
  args.v = v_cache.data_ptr();
  args.tables = tables.data_ptr<int>();
  args.positions = positions.data_ptr<int>();
  args.out = out.data_ptr();
  args.batch = q.size(0);
  args.tokens = q.size(1);
  args.heads = q.size(2);
  args.dim = q.size(3);
  args.pages = k_cache.size(0);
  args.kv_heads = k_cache.size(1);
  args.page = k_cache.size(2);
  args.page_shift = __builtin_ctz(args.page);
  args.width = tables.size(1);
  args.scale_log2 = static_cast<float>(paged::kLog2e / std::sqrt(static_cast<double>(args.dim)));
  auto stream = at::cuda::getCurrentCUDAStream();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  if (rows_path(q, k_cache, v_cache)) {
    if (q.scalar_type() == at::kHalf) paged_rows_launch<__half>(args, sms, stream);
    else paged_rows_launch<__nv_bfloat16>(args, sms, stream);
    return out;
  }
  switch (q.scalar_type()) {
    case at::kFloat: paged_simt_launch<float>(args, sms, stream); break;
    case at::kHalf: paged_simt_launch<__half>(args, sms, stream); break;
    case at::kBFloat16: paged_simt_launch<__nv_bfloat16>(args, sms, stream); break;
    default: TORCH_CHECK(false, "paged_attention: fp32, fp16 or bf16");
  }
  return out;
}

}  // namespace eb
