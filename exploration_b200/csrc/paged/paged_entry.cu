// Entry point of paged_attention: argument block and choice of kernel.
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>

#include "paged_checks.h"
#include "paged_launch.h"

namespace eb {

using paged::Args;

namespace {

enum class Path { kCudaCore, kTileFp32, kRows, kChunk };

// The kernel of a call. Head dims 64 and 128 (one or two 128-byte swizzle spans of
// a 16-bit type) have kernels of their own: up to 16 rows of a key head are bound
// by the read of the cache, more by arithmetic. Measured with four sequences over
// 30,000 keys, 16 heads of 64:
//   bf16, few-row / chunk kernel: 8 rows 86 / 98 us, 16 rows 90 / 100, 17 rows 157
//     (keys read twice) / 99; over 500 keys 16 rows 14 / 21;
//   fp32, general / tiled kernel: 2 rows 219 / 363 us, 4 rows 304 / 363, 5 rows
//     352 / 364, 6 rows 402 / 363, 12 rows 941 / 365.
// Five rows are a tie; 8 key heads of 128 give 233 / 399 us for 2 rows and 381 / 396 for 5.
// Over a few hundred keys the tiles win from fewer rows on (4 rows of 8 key heads of
// 128 over 500 keys: 41 / 20 us), which the rule does not use: the host does not know lengths.
Path choose(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache) {
  const int64_t dim = q.size(3);
  auto aligned = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; };
  const bool q_aligned = !q.is_contiguous() || aligned(q);   // strided queries are copied first
  if ((dim != 64 && dim != 128) || !q_aligned || !aligned(k_cache) || !aligned(v_cache)) return Path::kCudaCore;
  const int64_t rows = q.size(1) * (q.size(2) / k_cache.size(1));
  if (q.scalar_type() == at::kFloat) return rows <= 4 ? Path::kCudaCore : Path::kTileFp32;
  return rows <= 16 ? Path::kRows : Path::kChunk;
}

template <typename T>
void launch(Path path, Args& args, int sms, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (path == Path::kRows) return paged_rows_launch<T>(args, sms, stream);
    if (path == Path::kChunk) return paged_chunk_launch<T>(args, sms, stream);
  } else {
    if (path == Path::kTileFp32) return paged_tile_fp32_launch(args, sms, stream);
  }
  paged_simt_launch<T>(args, sms, stream);
}

}  // namespace

std::string paged_attention_path(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache) {
  const Path path = choose(q, k_cache, v_cache);
  switch (path) {
    case Path::kRows: return "rows";
    case Path::kChunk: return "tcgen05";
    case Path::kTileFp32: return "fp32_tile";
    default: return "cuda_core";
  }
}

at::Tensor paged_attention(const at::Tensor& q_in, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& tables_in, const at::Tensor& positions_in) {
  paged::check_cache(q_in, k_cache, v_cache, tables_in, positions_in);
  c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = q_in.contiguous(), tables = tables_in.contiguous(), positions = paged::int32(positions_in);
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
  const uintptr_t four = 4 * q.element_size();
  args.vectors = args.dim % 4 == 0 && reinterpret_cast<uintptr_t>(args.q) % four == 0 &&
                 reinterpret_cast<uintptr_t>(args.k) % four == 0 && reinterpret_cast<uintptr_t>(args.v) % four == 0;
  args.scale_log2 = static_cast<float>(paged::kLog2e / std::sqrt(static_cast<double>(args.dim)));
  auto stream = at::cuda::getCurrentCUDAStream();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const Path path = choose(q, k_cache, v_cache);
  switch (q.scalar_type()) {
    case at::kFloat: launch<float>(path, args, sms, stream); break;
    case at::kHalf: launch<__half>(path, args, sms, stream); break;
    case at::kBFloat16: launch<__nv_bfloat16>(path, args, sms, stream); break;
    default: TORCH_CHECK(false, "paged_attention: fp32, fp16 or bf16");
  }
  return out;
}

}  // namespace eb
