// Joins the partial results of the paged-attention kernels.
//
// An item (entry, head) that was cut into runs left, for every row, a maximum
// m_i, a sum l_i and a vector o_i = sum 2^(a - m_i) v of each part. With
// m = max m_i the result is sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, the
// parts taken in key order.
//
// A column of CTAs looks at the cut at the start of its run: if it is the first
// one inside its item, the item's parts are those of the run before, this one
// and so on up to the item's end. Bound by latency: the parts were just written
// and sit in L2. The launch overlaps the attention kernel's tail (programmatic
// dependent launch).
#include <ATen/ATen.h>

#include <algorithm>

#include "paged_common.cuh"

namespace eb {
namespace {

using namespace paged;

// The cut at the start of run blockIdx.x + 1, when it is the first inside its item.
struct Cut {
  int run, begin, parts, entry, head, rows, token0, batch;

  EB_DEVICE bool read(const Args& p) {
    const int c = blockIdx.x + 1;
    const int4 cut = reinterpret_cast<const int4*>(p.cuts)[c];
    run = *p.run;
    begin = cut.z;
    if (begin == 0 || begin > run) return false;   // no cut inside an item, or not its first
    parts = 1 + (cut.w - begin + run - 1) / run;
    entry = cut.x;
    head = cut.y;
    batch = entry / p.row_tiles;
    token0 = (entry - batch * p.row_tiles) * p.tile_tokens;
    rows = min(p.tile_tokens, p.tokens - token0) * p.group;
    return true;
  }

  // Partial slot of part i: the last item of run c - 1 (its first one when it is the only one), then
  // the first items of the runs that follow.
  EB_DEVICE int64_t slot(int i) const {
    const int64_t c = blockIdx.x + 1;
    return i == 0 ? 2 * (c - 1) + (begin == run ? 0 : 1) : 2 * (c - 1 + i);
  }

  EB_DEVICE int64_t out_row(const Args& p, int row) const {
    return (static_cast<int64_t>(batch) * p.tokens + token0 + row / p.group) * p.heads + head * p.group +
           row % p.group;
  }
};

constexpr int kMaxElems = 8;   // elements of a row a lane holds (head dims up to 256)

// Few rows, perhaps many parts: a CTA of four warps a row, the parts dealt to the warps.
template <typename T>
__global__ void __launch_bounds__(128)
paged_combine_row_kernel(Args p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm_o[4][256];
  __shared__ float sm_ml[4][2];
  Cut cut;
  if (!cut.read(p)) return;
  const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (row >= cut.rows) return;
  float m = kNegInf, sum = 0.f, acc[kMaxElems];
#pragma unroll
  for (int i = 0; i < kMaxElems; ++i) acc[i] = 0.f;
  // This warp's parts, up to 32 at a time: factors first, one a lane, then the vectors.
  for (int base = 0; base * 4 < cut.parts; base += 32) {
    const int mine = (base + lane) * 4 + warp;
    float2 ml = make_float2(kNegInf, 0.f);   // also what a part without keys holds
    if (mine < cut.parts) ml = *reinterpret_cast<const float2*>(p.part_ml + (cut.slot(mine) * p.row_tile + row) * 2);
    const float next = fmaxf(m, warp_max(ml.x)), ref = finite_or_zero(next);
    const float keep = ex2(m - ref), f = ex2(ml.x - ref);
    m = next;
    sum = sum * keep + warp_sum(f * ml.y);
#pragma unroll
    for (int i = 0; i < kMaxElems; ++i) acc[i] *= keep;
    const int count = min(32, (cut.parts - warp - base * 4 + 3) / 4);
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const float* o = p.part_o + (cut.slot((base + j) * 4 + warp) * p.row_tile + row) * p.dim;
      const float w = __shfl_sync(0xffffffffu, f, j);
#pragma unroll
      for (int i = 0; i < kMaxElems; ++i)
        if (lane + 32 * i < p.dim) acc[i] = fmaf(w, o[lane + 32 * i], acc[i]);
    }
  }
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
  T* dst = static_cast<T*>(p.out) + cut.out_row(p, row) * p.dim;
  for (int d = threadIdx.x; d < p.dim; d += blockDim.x) {
    float total = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = ex2(sm_ml[w][0] - ref);
      total += f * sm_ml[w][1];
      x = fmaf(f, sm_o[w][d], x);
    }
    dst[d] = cast_f<T>(total == 0.f ? 0.f : x / total);
  }
}

// Many rows, mostly two or three parts: a thread takes four elements of a row.
template <typename T>
__global__ void __launch_bounds__(256)
paged_combine_rows_kernel(Args p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Cut cut;
  if (!cut.read(p)) return;
  const int quads = p.dim / 4;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < cut.rows * quads; i += gridDim.y * blockDim.x) {
    const int row = i / quads, d = (i - row * quads) * 4;
    float m = kNegInf, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int part = 0; part < cut.parts; ++part) {
      const int64_t at = cut.slot(part) * p.row_tile + row;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
      const float4 o = *reinterpret_cast<const float4*>(p.part_o + at * p.dim + d);
      const float next = fmaxf(m, ml.x), ref = finite_or_zero(next);
      const float keep = ex2(m - ref), f = ex2(ml.x - ref);
      m = next;
      sum = sum * keep + f * ml.y;
      acc.x = acc.x * keep + f * o.x;
      acc.y = acc.y * keep + f * o.y;
      acc.z = acc.z * keep + f * o.z;
      acc.w = acc.w * keep + f * o.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* dst = static_cast<T*>(p.out) + cut.out_row(p, row) * p.dim + d;
    dst[0] = cast_f<T>(acc.x * inv);
    dst[1] = cast_f<T>(acc.y * inv);
    dst[2] = cast_f<T>(acc.z * inv);
    dst[3] = cast_f<T>(acc.w * inv);
  }
}

}  // namespace

template <typename T>
void paged_combine_launch(const Args& args, int ctas, cudaStream_t stream) {
  const int rows = args.row_tile;
  cudaLaunchConfig_t config = {};
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  // The many-row form reads 16-byte vectors: more than 16 rows of an item come from the chunk
  // kernel and the fp32 tiles only, whose head dims are 64 and 128.
  if (rows <= 16) {
    config.gridDim = dim3(ctas - 1, rows);
    config.blockDim = dim3(128);
    EB_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_combine_row_kernel<T>, args));
  } else {
    TORCH_CHECK(args.dim % 4 == 0, "paged_attention: many-row items need head dims of whole vectors");
    config.gridDim = dim3(ctas - 1, std::min(16, cdiv(rows * args.dim / 4, 256)));
    config.blockDim = dim3(256);
    EB_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_combine_rows_kernel<T>, args));
  }
  count_launch(1);
}

template void paged_combine_launch<float>(const Args&, int, cudaStream_t);
template void paged_combine_launch<__half>(const Args&, int, cudaStream_t);
template void paged_combine_launch<__nv_bfloat16>(const Args&, int, cudaStream_t);

}  // namespace eb
