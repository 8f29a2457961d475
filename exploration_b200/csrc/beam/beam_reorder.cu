// Reordering of a paged cache after a selection: new tables, and a copy of the
// partly filled page of every beam that takes over another beam's state.
//
// The beams of a group have the same length n. Full pages (j < n / page) are
// never written again, so beam i's new table names its parent's pages there.
// The page being filled is private to a beam: when the parent is another beam,
// its first n % page rows are copied, in every layer and head, into beam i's
// spare page, which takes that page's place in the table while the old page
// becomes the spare. Copies read pages of the old tables and write spare pages
// only, so no beam reads what another one writes and the CTAs need no order.
//
// Bound by memory: the filled rows of the copied pages, read and written once
// with 16-byte vectors, four in flight a thread. One CTA takes a few heads of one
// (beam, layer, keys or values); the first one of a beam also writes its tables.
// Measured: 24 beams, 12 layers of 16 heads of 64, pages of 64 about 45 rows full
// (72 MB): 14.4 us of kernel, 5.0 TB/s; 20.4 us with all heads in one CTA.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "../common/checks.h"
#include "../common/util.cuh"

namespace eb {
namespace {

struct ReorderArgs {
  char* k;                 // [layers, pages, kv_heads, page, row bytes]
  char* v;
  const int* tables;       // [groups, beams, width]
  const int* spare;        // [groups, beams]
  const int64_t* parents;
  const int* lengths;      // [groups]
  int* tables_out;
  int* spare_out;
  int64_t layer_bytes, page_bytes, head_bytes;
  int beams, width, pages, kv_heads, page, row_bytes, heads_per_cta;
};

template <typename V>
__global__ void __launch_bounds__(256)
beam_reorder_kernel(ReorderArgs p) {
  const int slot = blockIdx.x, group = slot / p.beams, beam = slot - group * p.beams;
  const int n = max(p.lengths[group], 0), tail = n / p.page, rows = n - tail * p.page;
  const int64_t wanted = p.parents[slot];
  const int parent = wanted >= 0 && wanted < p.beams ? static_cast<int>(wanted) : beam;
  const int* mine = p.tables + static_cast<int64_t>(slot) * p.width;
  const int* theirs = p.tables + static_cast<int64_t>(group * p.beams + parent) * p.width;
  const bool moves = parent != beam && rows > 0 && tail < p.width;
  const int fresh = p.spare[slot];
  if (blockIdx.y == 0 && blockIdx.z == 0) {
    int* out = p.tables_out + static_cast<int64_t>(slot) * p.width;
    for (int j = threadIdx.x; j < p.width; j += blockDim.x)
      out[j] = j < tail ? theirs[j] : (moves && j == tail ? fresh : mine[j]);
    if (threadIdx.x == 0) p.spare_out[slot] = moves ? mine[tail] : fresh;
  }
  if (!moves) return;
  const int from = theirs[tail];
  // Also the end of a call on empty pools, which have no page.
  if (from < 0 || from >= p.pages || fresh < 0 || fresh >= p.pages) return;
  char* cache = (blockIdx.y & 1 ? p.v : p.k) + (blockIdx.y >> 1) * p.layer_bytes;
  const char* src = cache + from * p.page_bytes;
  char* dst = cache + fresh * p.page_bytes;
  // The heads of this CTA: each a contiguous span of `rows` rows.
  const int h0 = blockIdx.z * p.heads_per_cta, heads = min(p.heads_per_cta, p.kv_heads - h0);
  src += h0 * p.head_bytes;
  dst += h0 * p.head_bytes;
  const int per_head = rows * (p.row_bytes / static_cast<int>(sizeof(V)));
  const int total = per_head * heads;
  auto place = [&](int i) {
    const int head = i / per_head;
    return head * p.head_bytes + static_cast<int64_t>(i - head * per_head) * sizeof(V);
  };
  constexpr int kUnroll = 4;
  const int step = blockDim.x * kUnroll;
  for (int base = threadIdx.x; base < total; base += step) {
    V x[kUnroll];
    int64_t at[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = base + u * blockDim.x;
      at[u] = i < total ? place(i) : -1;
      if (at[u] >= 0) x[u] = *reinterpret_cast<const V*>(src + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (at[u] >= 0) *reinterpret_cast<V*>(dst + at[u]) = x[u];
  }
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> beam_reorder(at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& tables_in,
                                                const at::Tensor& spare_in, const at::Tensor& parents_in,
                                                const at::Tensor& lengths_in) {
  // The Python module makes the same checks for CPU tensors, with the same messages.
  TORCH_CHECK_VALUE(k_cache.dim() == 5 && k_cache.sizes() == v_cache.sizes() && tables_in.dim() == 3 &&
                        spare_in.dim() == 2 && spare_in.size(0) == tables_in.size(0) &&
                        spare_in.size(1) == tables_in.size(1) && parents_in.sizes() == spare_in.sizes() &&
                        lengths_in.dim() == 1 && lengths_in.size(0) == spare_in.size(0) && tables_in.size(2) >= 1,
                    "expected pools [layers, pages, kv_heads, page, head_dim], tables [groups, beams, width], "
                    "spare, parents [groups, beams] and lengths [groups]");
  TORCH_CHECK_VALUE(k_cache.size(3) >= 1, "a page must hold at least one token");
  TORCH_CHECK_VALUE(k_cache.scalar_type() == v_cache.scalar_type() && k_cache.element_size() % 2 == 0,
                    "key and value pools must have one dtype of 16 bits or more");
  TORCH_CHECK_VALUE(tables_in.scalar_type() == at::kInt && spare_in.scalar_type() == at::kInt &&
                        lengths_in.scalar_type() == at::kInt && parents_in.scalar_type() == at::kLong,
                    "tables, spare and lengths must be int32 and parents int64");
  TORCH_CHECK_VALUE(same_device(k_cache, v_cache, tables_in, spare_in, parents_in, lengths_in),
                    "all tensors must be on one device");
  TORCH_CHECK_VALUE(k_cache.is_contiguous() && v_cache.is_contiguous(), "cache pools must be contiguous");
  TORCH_CHECK_VALUE(!wants_grad(k_cache) && !wants_grad(v_cache), "beam_reorder is for inference: it has no gradient");
  c10::cuda::CUDAGuard guard(k_cache.device());
  const at::Tensor tables = tables_in.contiguous(), spare = spare_in.contiguous(), parents = parents_in.contiguous(),
                   lengths = lengths_in.contiguous();
  at::Tensor tables_out = at::empty_like(tables), spare_out = at::empty_like(spare);
  const int64_t slots = spare.numel(), layers = k_cache.size(0);
  if (slots == 0) return {tables_out, spare_out};
  TORCH_CHECK(layers < 32768, "beam_reorder: too many layers");
  const int64_t row_bytes = k_cache.size(4) * k_cache.element_size();
  ReorderArgs args{};
  args.k = static_cast<char*>(k_cache.data_ptr());
  args.v = static_cast<char*>(v_cache.data_ptr());
  args.tables = tables.data_ptr<int>();
  args.spare = spare.data_ptr<int>();
  args.parents = parents.data_ptr<int64_t>();
  args.lengths = lengths.data_ptr<int>();
  args.tables_out = tables_out.data_ptr<int>();
  args.spare_out = spare_out.data_ptr<int>();
  args.kv_heads = k_cache.size(2);
  args.page = k_cache.size(3);
  args.row_bytes = row_bytes;
  args.head_bytes = args.page * row_bytes;
  args.page_bytes = args.kv_heads * args.head_bytes;
  // Pools without an element (no layers, heads, elements or pages) have nothing to copy: the tables alone are written.
  const bool copies = k_cache.numel() > 0;
  args.pages = copies ? k_cache.size(1) : 0;
  args.layer_bytes = args.pages * args.page_bytes;
  args.beams = spare.size(1);
  args.width = tables.size(2);
  // Heads of a CTA: about 16 KB of a full page, all of it in flight at once.
  dim3 grid(slots);
  if (copies) {
    args.heads_per_cta = std::max<int64_t>(1, std::min<int64_t>(args.kv_heads, 16384 / args.head_bytes));
    grid = dim3(slots, 2 * layers, cdiv(args.kv_heads, args.heads_per_cta));
  }
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool wide = row_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(args.k) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(args.v) % 16 == 0;
  if (wide) beam_reorder_kernel<uint4><<<grid, 256, 0, stream>>>(args);
  else beam_reorder_kernel<uint16_t><<<grid, 256, 0, stream>>>(args);
  EB_CUDA_CHECK(cudaGetLastError());
  count_launch(1);
  return {tables_out, spare_out};
}

}  // namespace eb
