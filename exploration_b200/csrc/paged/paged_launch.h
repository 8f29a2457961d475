// Host side of the paged-attention kernels: row tiles, split and workspace.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "../common/tma.cuh"
#include "paged_common.cuh"

namespace eb {
namespace paged {

// The pool [pages * kv_heads, page, dim] of a 16-bit type for TMA loads of one
// plane's `rows` x 64 boxes (at most a page), 128-byte swizzle. Planes past the
// pool read as zero.
inline CUtensorMap make_pool_map(const Args& args, const void* base, bool half, int rows) {
  bind_primary_context();
  TORCH_CHECK(reinterpret_cast<uintptr_t>(base) % 16 == 0, "paged_attention: pools must be 16-byte aligned");
  const int64_t planes = static_cast<int64_t>(args.pages) * args.kv_heads;
  TORCH_CHECK(planes < (1LL << 31) - 1, "paged_attention: too many pages");
  CUtensorMap map;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(args.dim), static_cast<cuuint64_t>(args.page),
                        static_cast<cuuint64_t>(planes)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(args.dim) * 2, static_cast<cuuint64_t>(args.page) * args.dim * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(std::min(args.page, rows)), 1};
  cuuint32_t unit[3] = {1, 1, 1};
  CUresult res = tensor_map_encoder()(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                      3, const_cast<void*>(base), dims, strides, box, unit,
                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with ", static_cast<int>(res));
  return map;
}

// The queries [batch, tokens, heads, dim] for TMA loads of one item's rows: `tokens`
// tokens of a group's heads (token by token), 128-byte swizzle. Tokens past the
// call's read as zero.
inline CUtensorMap make_query_map(const Args& args, bool half, int tokens) {
  bind_primary_context();
  TORCH_CHECK(reinterpret_cast<uintptr_t>(args.q) % 16 == 0, "paged_attention: queries must be 16-byte aligned");
  CUtensorMap map;
  const cuuint64_t row = static_cast<cuuint64_t>(args.dim) * 2;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(args.dim), static_cast<cuuint64_t>(args.heads),
                        static_cast<cuuint64_t>(args.tokens), static_cast<cuuint64_t>(args.batch)};
  cuuint64_t strides[3] = {row, row * args.heads, row * args.heads * args.tokens};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(args.group), static_cast<cuuint32_t>(tokens), 1};
  cuuint32_t unit[4] = {1, 1, 1, 1};
  CUresult res = tensor_map_encoder()(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                      4, const_cast<void*>(args.q), dims, strides, box, unit,
                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with ", static_cast<int>(res));
  return map;
}

// Lets a kernel use `bytes` of dynamic shared memory, once per kernel and device.
inline void allow_smem(const void* kernel, size_t bytes) {
  static std::mutex mutex;
  static std::set<std::pair<const void*, int>> done;
  std::lock_guard<std::mutex> lock(mutex);
  if (done.insert({kernel, at::cuda::current_device()}).second)
    EB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
}

// Row tiles of at most `most` rows: whole tokens of a group; a group that is
// larger is divided into equal parts, each an item of its own.
inline void set_rows(Args& args, int most, int key_tile) {
  const int whole = args.heads / args.kv_heads;
  int part = whole;
  while (part > most || whole % part) --part;
  args.group = part;
  args.head_div = whole / part;
  args.item_heads = args.kv_heads * args.head_div;
  args.tile_tokens = std::min(args.tokens, std::max(1, most / part));
  args.row_tile = args.tile_tokens * part;
  args.row_tiles = cdiv(args.tokens, args.tile_tokens);
  args.key_tile = key_tile;
}

// The split of one call: CTAs, and the workspace of the cut items. The
// workspace comes from the stream-ordered caching allocator and is given back
// when the call has been enqueued.
struct Split {
  int ctas = 0;
  at::Tensor space;

  // `whole_tiles`: items of at most so many key tiles are not cut. `item_cost`: see Args.
  Split(Args& args, int wanted, int whole_tiles, int item_cost) {
    const int64_t entries = static_cast<int64_t>(args.batch) * args.row_tiles;
    const int64_t items = entries * args.item_heads;
    const int64_t longest = cdiv64(static_cast<int64_t>(args.width) * args.page, args.key_tile);
    args.item_cost = item_cost;
    args.flat = entries <= kMaxEntries && longest > whole_tiles && items * (longest + item_cost) < (1LL << 31);
    if (!args.flat) {
      TORCH_CHECK(items < (1LL << 31), "paged_attention: too many rows");
      ctas = static_cast<int>(items);
      return;
    }
    ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(wanted, items * longest)));
    // One allocation: partial vectors, statistics, cuts.
    const int64_t rows = 2LL * ctas * args.row_tile;
    space = at::empty({rows * (args.dim + 2) + 4LL * ctas + 1},
                      at::TensorOptions().device(at::kCUDA, at::cuda::current_device()).dtype(at::kFloat));
    args.cuts = reinterpret_cast<int*>(space.data_ptr<float>());   // 16-byte entries first
    args.part_o = space.data_ptr<float>() + 4LL * ctas;
    args.part_ml = args.part_o + rows * args.dim;
    args.run = reinterpret_cast<int*>(args.part_ml + rows * 2);
  }

  static int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

  template <typename T>
  void combine(const Args& args, cudaStream_t stream) const {
    if (args.flat && ctas > 1) paged_combine_launch<T>(args, ctas, stream);
  }
};

}  // namespace paged

template <typename T>
void paged_simt_launch(paged::Args& args, int sms, cudaStream_t stream);
template <typename T>
void paged_rows_launch(paged::Args& args, int sms, cudaStream_t stream);
template <typename T>
void paged_chunk_launch(paged::Args& args, int sms, cudaStream_t stream);
void paged_tile_fp32_launch(paged::Args& args, int sms, cudaStream_t stream);

}  // namespace eb
