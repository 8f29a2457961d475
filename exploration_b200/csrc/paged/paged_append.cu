// Appending new tokens to a paged cache, with the position rotation on the way.
//
// For a token at position p, with c = cos[p], s = sin[p] and the halves x1, x2
// of a head: y1 = x1 c - x2 s, y2 = x2 c + x1 s in fp32, rounded once. Queries
// go to a dense tensor, keys and values to row p % page of pool page
// tables[b, p / page]. A position of -1 (or one outside the table or the
// rotation tables) writes nothing and leaves zero queries.
//
// Bound by memory: every element is read and written once, and the D floats of
// a token's rotation row are shared by all heads through L1. One CTA takes one
// token, so position, page and rotation row are looked up once; a thread takes
// one 16-byte vector of the first half of a head and its partner in the second.
// Measured: 4,245 tokens in 4 x 2,011 rows, 32 + 2 x 8 heads of 128, bf16 (138 MB): 25.5 us of
// kernel, 5.4 TB/s. CTAs of 384 threads (a vector pair each, 33 us) and loads begun
// before the position is known (32.6 us) were slower.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "../common/util.cuh"
#include "paged_checks.h"

namespace eb {
namespace {

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* cos;
  const float* sin;
  const int* tables;
  const int* positions;
  void* q_out;
  void* k_cache;
  void* v_cache;
  int64_t qs[3], ks[3], vs[3];   // strides of batch, token and head
  int tokens, heads, kv_heads, dim, width, pages, page, page_shift, rows;   // rows: of cos / sin
};

template <typename T, int VE>
struct alignas(sizeof(T) * VE) Vec {
  T x[VE];
};

template <typename T, int VE>
__global__ void __launch_bounds__(128)
paged_append_kernel(AppendArgs p) {
  using V = Vec<T, VE>;
  const int64_t token = blockIdx.x;
  const int b = static_cast<int>(token / p.tokens), t = static_cast<int>(token - static_cast<int64_t>(b) * p.tokens);
  const int pos = p.positions[token];
  const int half = p.dim / 2, per_head = half / VE;
  int id = -1;
  if (pos >= 0 && pos < p.rows && (pos >> p.page_shift) < p.width)
    id = p.tables[static_cast<int64_t>(b) * p.width + (pos >> p.page_shift)];
  const bool real = id >= 0 && id < p.pages;
  const int units = (p.heads + (real ? 2 * p.kv_heads : 0)) * per_head;
  const int64_t row = pos & (p.page - 1);
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    int head = u / per_head;
    const int d = (u - head * per_head) * VE;
    const T* src;
    T* dst;
    bool turn = true;
    if (head < p.heads) {
      src = static_cast<const T*>(p.q) + b * p.qs[0] + t * p.qs[1] + head * p.qs[2];
      dst = static_cast<T*>(p.q_out) + (token * p.heads + head) * p.dim;
    } else {
      head -= p.heads;
      turn = head < p.kv_heads;
      if (!turn) head -= p.kv_heads;
      const int64_t* st = turn ? p.ks : p.vs;
      src = static_cast<const T*>(turn ? p.k : p.v) + b * st[0] + t * st[1] + head * st[2];
      dst = static_cast<T*>(turn ? p.k_cache : p.v_cache) +
            ((static_cast<int64_t>(id) * p.kv_heads + head) * p.page + row) * p.dim;
    }
    V first, second;
    if (!real) {
#pragma unroll
      for (int i = 0; i < VE; ++i) first.x[i] = second.x[i] = cast_f<T>(0.f);
    } else {
      first = *reinterpret_cast<const V*>(src + d);
      second = *reinterpret_cast<const V*>(src + half + d);
      if (turn) {
        const float* c = p.cos + static_cast<int64_t>(pos) * half + d;
        const float* s = p.sin + static_cast<int64_t>(pos) * half + d;
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float x1 = load_f<T>(&first.x[i]), x2 = load_f<T>(&second.x[i]);
          first.x[i] = cast_f<T>(x1 * c[i] - x2 * s[i]);
          second.x[i] = cast_f<T>(x2 * c[i] + x1 * s[i]);
        }
      }
    }
    *reinterpret_cast<V*>(dst + d) = first;
    *reinterpret_cast<V*>(dst + half + d) = second;
  }
}

template <typename T>
void launch(const AppendArgs& args, int64_t count, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  bool wide = args.dim % (2 * kWide) == 0 && aligned(args.q) && aligned(args.k) && aligned(args.v) &&
              aligned(args.q_out) && aligned(args.k_cache) && aligned(args.v_cache);
  for (int i = 0; i < 3; ++i)
    wide = wide && args.qs[i] % kWide == 0 && args.ks[i] % kWide == 0 && args.vs[i] % kWide == 0;
  if (wide) paged_append_kernel<T, kWide><<<count, 128, 0, stream>>>(args);
  else paged_append_kernel<T, 1><<<count, 128, 0, stream>>>(args);
  EB_CUDA_CHECK(cudaGetLastError());
  count_launch(1);
}

}  // namespace

at::Tensor paged_append(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                        const at::Tensor& cos_in, const at::Tensor& sin_in, at::Tensor& k_cache, at::Tensor& v_cache,
                        const at::Tensor& tables_in, const at::Tensor& positions_in) {
  paged::check_cache(q_in, k_cache, v_cache, tables_in, positions_in);
  TORCH_CHECK_VALUE(k_in.sizes() == v_in.sizes() && k_in.dim() == 4 && k_in.size(0) == q_in.size(0) &&
                        k_in.size(1) == q_in.size(1) && k_in.size(2) == k_cache.size(1) && k_in.size(3) == q_in.size(3),
                    "expected k, v [batch, tokens, kv_heads, head_dim]");
  TORCH_CHECK_VALUE(k_in.scalar_type() == q_in.scalar_type() && v_in.scalar_type() == q_in.scalar_type() &&
                        same_device(q_in, k_in, v_in, cos_in, sin_in),
                    "queries, keys, values and rotation tables must match in dtype and device");
  TORCH_CHECK_VALUE(cos_in.sizes() == sin_in.sizes() && cos_in.dim() == 2 && cos_in.size(1) * 2 == q_in.size(3) &&
                        cos_in.scalar_type() == at::kFloat && sin_in.scalar_type() == at::kFloat,
                    "expected fp32 cos, sin [positions, head_dim / 2]");
  TORCH_CHECK_VALUE(!wants_grad(k_in) && !wants_grad(v_in) && !wants_grad(cos_in) && !wants_grad(sin_in),
                    "paged operators are for inference: they have no gradient");
  c10::cuda::CUDAGuard guard(q_in.device());
  auto rows = [](const at::Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); };
  const at::Tensor q = rows(q_in), k = rows(k_in), v = rows(v_in), cos = cos_in.contiguous(), sin = sin_in.contiguous();
  const at::Tensor tables = tables_in.contiguous(), positions = paged::int32(positions_in);
  const int64_t batch = q.size(0), tokens = q.size(1), heads = q.size(2), dim = q.size(3);
  at::Tensor out = at::empty({batch, tokens, heads, dim}, q.options());
  if (batch * tokens == 0) return out;
  TORCH_CHECK(batch * tokens < (1LL << 31), "paged_append: too many tokens");
  AppendArgs args{};
  args.q = q.data_ptr();
  args.k = k.data_ptr();
  args.v = v.data_ptr();
  args.cos = cos.data_ptr<float>();
  args.sin = sin.data_ptr<float>();
  args.tables = tables.data_ptr<int>();
  args.positions = positions.data_ptr<int>();
  args.q_out = out.data_ptr();
  args.k_cache = k_cache.data_ptr();
  args.v_cache = v_cache.data_ptr();
  for (int i = 0; i < 3; ++i) {
    args.qs[i] = q.stride(i);
    args.ks[i] = k.stride(i);
    args.vs[i] = v.stride(i);
  }
  args.tokens = tokens;
  args.heads = heads;
  args.kv_heads = k.size(2);
  args.dim = dim;
  args.width = tables.size(1);
  args.pages = k_cache.size(0);
  args.page = k_cache.size(2);
  args.page_shift = __builtin_ctz(args.page);
  args.rows = cos.size(0);
  auto stream = at::cuda::getCurrentCUDAStream();
  switch (q.scalar_type()) {
    case at::kFloat: launch<float>(args, batch * tokens, stream); break;
    case at::kHalf: launch<__half>(args, batch * tokens, stream); break;
    case at::kBFloat16: launch<__nv_bfloat16>(args, batch * tokens, stream); break;
    default: TORCH_CHECK(false, "paged_append: fp32, fp16 or bf16");
  }
  return out;
}

}  // namespace eb
