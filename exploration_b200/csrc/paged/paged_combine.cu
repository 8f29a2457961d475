// Joins the partial results of the paged-attention kernels.
//
// An item (entry, head) that was cut into runs left, for every row, a maximum
// m_i, a sum l_i and a vector o_i = sum 2^(a - m_i) v of each part. With
// m = max m_i the result is sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, the
// parts taken in key order.
//
// CTA column c looks at the cut at the start of run c: if it is the first one
// inside its item, the item's parts are those of runs c - 1, c, ... up to the
// item's end. Bound by latency: the parts were just written and sit in L2. One
// warp joins a row; four share it where rows are few and parts may be many. The
// launch overlaps the attention kernel's tail (programmatic dependent launch).
#include <ATen/ATen.h>

#include "paged_common.cuh"

namespace eb {
namespace {

using namespace paged;

constexpr int kMaxElems = 8;   // elements of a row a lane holds (head dims up to 256)

template <typename T>
__global__ void __launch_bounds__(128)
paged_combine_kernel(Args p, int rows_per_cta, int warps_per_row) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm_o[4][256];
  __shared__ float sm_ml[4][2];
  const int c = blockIdx.x + 1;
  const int4 cut = reinterpret_cast<const int4*>(p.cuts)[c];
  const int run = *p.run, begin = cut.z, tiles = cut.w;
  if (begin == 0 || begin > run) return;   // no cut inside an item, or not its first
  const int parts = 1 + (tiles - begin + run - 1) / run;
  auto slot = [&](int i) { return i == 0 ? 2LL * (c - 1) + (begin == run ? 0 : 1) : 2LL * (c - 1 + i); };
  const int entry = cut.x, head = cut.y;
  const int batch = entry / p.row_tiles, token0 = (entry - batch * p.row_tiles) * p.tile_tokens;
  const int rows = min(p.tile_tokens, p.tokens - token0) * p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = warps_per_row == 4 ? warp : 0;
  const int end = min(rows, (static_cast<int>(blockIdx.y) + 1) * rows_per_cta);
  for (int row = blockIdx.y * rows_per_cta + (warps_per_row == 4 ? 0 : warp); row < end;
       row += warps_per_row == 4 ? 1 : 4) {
    float m = kNegInf, sum = 0.f, acc[kMaxElems];
#pragma unroll
    for (int i = 0; i < kMaxElems; ++i) acc[i] = 0.f;
    // This warp's parts, up to 32 at a time: factors first, one a lane, then the vectors.
    for (int base = 0; base * warps_per_row < parts; base += 32) {
      const int mine = (base + lane) * warps_per_row + first;
      float2 ml = make_float2(kNegInf, 0.f);   // also what a part without keys holds
      if (mine < parts) ml = *reinterpret_cast<const float2*>(p.part_ml + (slot(mine) * p.row_tile + row) * 2);
      const float next = fmaxf(m, warp_max(ml.x)), ref = finite_or_zero(next);
      const float keep = ex2(m - ref), f = ex2(ml.x - ref);
      m = next;
      sum = sum * keep + warp_sum(f * ml.y);
#pragma unroll
      for (int i = 0; i < kMaxElems; ++i) acc[i] *= keep;
      const int count = min(32, (parts - first - base * warps_per_row + warps_per_row - 1) / warps_per_row);
#pragma unroll 4
      for (int j = 0; j < count; ++j) {
        const float* o = p.part_o + (slot((base + j) * warps_per_row + first) * p.row_tile + row) * p.dim;
        const float w = __shfl_sync(0xffffffffu, f, j);
#pragma unroll
        for (int i = 0; i < kMaxElems; ++i)
          if (lane + 32 * i < p.dim) acc[i] = fmaf(w, o[lane + 32 * i], acc[i]);
      }
    }
    if (warps_per_row == 4) {
      if (lane == 0) {
        sm_ml[warp][0] = m;
        sm_ml[warp][1] = sum;
      }
#pragma unroll
      for (int i = 0; i < kMaxElems; ++i)
        if (lane + 32 * i < p.dim) sm_o[warp][lane + 32 * i] = acc[i];
      __syncthreads();
      m = fmaxf(fmaxf(sm_ml[0][0], sm_ml[1][0]), fmaxf(sm_ml[2][0], sm_ml[3][0]));
      const float ref = finite_or_zero(m);
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < kMaxElems; ++i) acc[i] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = ex2(sm_ml[w][0] - ref);
        sum += f * sm_ml[w][1];
#pragma unroll
        for (int i = 0; i < kMaxElems; ++i)
          if (lane + 32 * i < p.dim) acc[i] = fmaf(f, sm_o[w][lane + 32 * i], acc[i]);
      }
      __syncthreads();
      if (warp != 0) continue;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int token = token0 + row / p.group, qhead = head * p.group + row % p.group;
    T* dst = static_cast<T*>(p.out) +
             ((static_cast<int64_t>(batch) * p.tokens + token) * p.heads + qhead) * p.dim;
#pragma unroll
    for (int i = 0; i < kMaxElems; ++i)
      if (lane + 32 * i < p.dim) dst[lane + 32 * i] = cast_f<T>(acc[i] * inv);
  }
}

}  // namespace

template <typename T>
void paged_combine_launch(const Args& args, int ctas, cudaStream_t stream) {
  // Few rows: a CTA a row. Many: a CTA takes 32 rows, eight a warp.
  const int rows = args.tile_tokens * args.group;
  const int per_cta = rows <= 16 ? 1 : 32, warps = rows <= 16 ? 4 : 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas - 1, cdiv(rows, per_cta));
  config.blockDim = dim3(128);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  EB_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_combine_kernel<T>, args, per_cta, warps));
  count_launch(1);
}

template void paged_combine_launch<float>(const Args&, int, cudaStream_t);
template void paged_combine_launch<__half>(const Args&, int, cudaStream_t);
template void paged_combine_launch<__nv_bfloat16>(const Args&, int, cudaStream_t);

}  // namespace eb
