// Joins the partial results of the paged-attention kernels.
//
// An item (entry, head) that was cut into runs left, for every row, a maximum
// m_i, a sum l_i and a vector o_i = sum 2^(a - m_i) v of each part. With
// m = max m_i the result is sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i; the
// parts are taken in key order. Items that one CTA finished are left alone;
// rows of an entry without keys become zero.
//
// Bound by latency: the partial sums were just written and sit in L2. The
// launch overlaps the attention kernel's tail (programmatic dependent launch).
#include <ATen/ATen.h>

#include "paged_common.cuh"

namespace eb {
namespace {

using namespace paged;

template <typename T>
__global__ void __launch_bounds__(128)
paged_combine_kernel(Args p, int ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int item = blockIdx.x;
  const int entry = item / p.item_heads, head = item - entry * p.item_heads;
  const int c0 = p.cum[entry], tiles = p.cum[entry + 1] - c0;
  const int64_t run = run_tiles(p, p.cum[p.batch * p.row_tiles], ctas);
  const int64_t a = static_cast<int64_t>(c0) * p.item_heads + static_cast<int64_t>(head) * tiles, b = a + tiles;
  const int first = static_cast<int>(a / run), last = tiles > 0 ? static_cast<int>((b - 1) / run) : first;
  if (tiles > 0 && first == last) return;
  const int batch = entry / p.row_tiles, token0 = (entry - batch * p.row_tiles) * p.tile_tokens;
  const int rows = min(p.tile_tokens, p.tokens - token0) * p.group;
  T* out = static_cast<T*>(p.out);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int row = blockIdx.y * 4 + warp; row < rows; row += gridDim.y * 4) {
    const int token = token0 + row / p.group, qhead = head * p.group + row % p.group;
    T* dst = out + ((static_cast<int64_t>(batch) * p.tokens + token) * p.heads + qhead) * p.dim;
    float m = kNegInf;
    if (tiles > 0) {
      for (int c = first + lane; c <= last; c += 32) {
        const int64_t slot = 2 * c + (c * run >= a ? 0 : 1);
        m = fmaxf(m, p.part_ml[(slot * p.row_tile + row) * 2]);
      }
      m = warp_max(m);
    }
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    float sum = 0.f;
    const float ref = finite_or_zero(m);   // a part without keys has m = -inf, l = 0, o = 0
    if (tiles > 0) {
      for (int c = first; c <= last; ++c) {
        const int64_t slot = 2 * c + (c * run >= a ? 0 : 1);
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (slot * p.row_tile + row) * 2);
        const float f = ex2(ml.x - ref);
        sum += f * ml.y;
        const float* o = p.part_o + (slot * p.row_tile + row) * p.dim;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (lane + 32 * i < p.dim) acc[i] += f * o[lane + 32 * i];
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.dim) dst[lane + 32 * i] = cast_f<T>(acc[i] * inv);
  }
}

}  // namespace

template <typename T>
void paged_combine_launch(const Args& args, int ctas, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  const int rows = args.tile_tokens * args.group;
  const int items = args.batch * args.row_tiles * args.item_heads;
  config.gridDim = dim3(items, rows > 16 ? cdiv(rows, 16) : cdiv(rows, 4));
  config.blockDim = dim3(128);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  EB_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_combine_kernel<T>, args, ctas));
  count_launch(1);
}

template void paged_combine_launch<float>(const Args&, int, cudaStream_t);
template void paged_combine_launch<__half>(const Args&, int, cudaStream_t);
template void paged_combine_launch<__nv_bfloat16>(const Args&, int, cudaStream_t);

}  // namespace eb
