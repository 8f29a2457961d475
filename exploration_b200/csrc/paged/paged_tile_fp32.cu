// Attention of new tokens over a paged cache in fp32 (head dim 64 or 128, more than
// four rows of a key head): IEEE fp32 products, no TF32.
//
// Bound by the fp32 pipe (75 TFLOP/s): every product comes from registers that
// 12 16-byte shared-memory loads fill for 128 multiply-adds. One CTA of 128
// threads takes 8 RPT rows (RPT 8, or 4 or 2 when there are no more) and walks
// 64-key tiles; a thread owns RPT rows x 4 keys of the scores and RPT rows x D / 16
// columns of the result, the 16 threads of a row
// sit in half a warp (row maxima and sums by shuffles). Weights go through
// shared memory, over the keys that they came from. Two or three CTAs an SM hide
// each other's loads. The products of a score are added from the last element to
// the first, one chain of fused multiply-adds.
//
// Measured: 64 tokens of four sequences over 9,000 keys, 32/8 heads of 128: 0.91 ms,
// 41 TFLOP/s (the general kernel, which shares a load between eight rows: 5.17 ms).
//
// Keys past an item's limit are masked and their values cleared on the way into
// shared memory: a page's unwritten rows may hold anything.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <climits>

#include "paged_common.cuh"
#include "paged_launch.h"

namespace eb {
namespace {

using namespace paged;

constexpr int kItemCost = 1;   // of an item's start and end, in tiles
constexpr int kTile = 64;
constexpr int kThreads = 128;

template <int D, int RPT>
struct TileSmem {
  static constexpr int kRows = 8 * RPT;
  static constexpr int kLd = D + 4;         // row pitch: eight rows reach all banks
  static constexpr int kLdW = kTile + 4;
  float q[kRows * kLd];
  float k[kTile * kLd];                     // then the weights [row][key]
  float v[kTile * D];
  Prefix table;
};

EB_DEVICE void copy16(float* dst, const float* src, bool real) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(real ? 16 : 0) : "memory");
}

EB_DEVICE void copies_done() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

// CTAs an SM, within registers (64 rows) and shared memory.
template <int D, int RPT>
constexpr int kCtas = D == 64 ? (RPT == 8 ? 3 : 4) : 2;

template <int D, int RPT>
__global__ void __launch_bounds__(kThreads, (kCtas<D, RPT>))
paged_tile_fp32_kernel(Args p) {
  extern __shared__ __align__(16) uint8_t raw[];
  using Smem = TileSmem<D, RPT>;
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  constexpr int kRows = Smem::kRows, kLd = Smem::kLd, kLdW = Smem::kLdW, kQuads = D / 4, kCols = D / 64;
  static_assert(kRows * kLdW <= kTile * kLd, "the weights fit over the keys");
  const int lane = threadIdx.x & 31, rg = threadIdx.x >> 4, cg = threadIdx.x & 15;
  float* weights = sm.k;
  if (p.flat) build_prefix(p, sm.table);
  Walk walk;
  walk.start(p, sm.table);
  publish_run<float>(p, sm.table, walk);
  Segment s;
  while (walk.next(p, sm.table, s)) {
    finish_segment(p, sm.table, s, lane);
    const int rows = min(p.tile_tokens, p.tokens - s.token0) * p.group;
    const int64_t row_base = static_cast<int64_t>(s.batch) * p.tokens + s.token0;
    auto query_row = [&](int r) {   // element offset of a row of the queries or the result
      return ((row_base + r / p.group) * p.heads + s.head * p.group + r % p.group) * D;
    };
    __syncthreads();   // the previous item's queries and weights have been read
    for (int i = threadIdx.x; i < kRows * kQuads; i += kThreads) {
      const int r = i / kQuads, d = (i % kQuads) * 4;
      copy16(&sm.q[r * kLd + d], static_cast<const float*>(p.q) + query_row(r < rows ? r : 0) + d, r < rows);
    }
    int pos[RPT], low = INT_MAX;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = rg * RPT + i;
      pos[i] = r < rows ? p.positions[row_base + r / p.group] : -1;
      if (pos[i] >= 0) low = min(low, pos[i]);
    }
    float o[RPT][4 * kCols], m[RPT], l[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      m[i] = kNegInf;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < 4 * kCols; ++c) o[i][c] = 0.f;
    }
    const int* table = p.tables + static_cast<int64_t>(s.batch) * p.width;
    const int kv_head = s.head / p.head_div;
    for (int tile = s.begin; tile < s.end; ++tile) {
      const int key0 = tile * kTile;
      __syncthreads();   // weights and values of the previous tile have been read
      for (int i = threadIdx.x; i < kTile * kQuads; i += kThreads) {
        const int r = i / kQuads, d = (i % kQuads) * 4, key = key0 + r;
        const int id = key < s.limit ? table[key >> p.page_shift] : -1;
        const bool real = id >= 0 && id < p.pages;
        const int64_t at =
            real ? ((static_cast<int64_t>(id) * p.kv_heads + kv_head) * p.page + (key & (p.page - 1))) * D + d : 0;
        copy16(&sm.k[r * kLd + d], static_cast<const float*>(p.k) + at, real);
        copy16(&sm.v[r * D + d], static_cast<const float*>(p.v) + at, real);
      }
      copies_done();
      __syncthreads();
      // Scores: rows rg * RPT + i, keys cg + 16 j.
      float a[RPT][4];
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) a[i][j] = 0.f;
#pragma unroll 2
      for (int d = D - 4; d >= 0; d -= 4) {
        float4 kx[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) kx[j] = *reinterpret_cast<const float4*>(&sm.k[(cg + 16 * j) * kLd + d]);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float4 qx = *reinterpret_cast<const float4*>(&sm.q[(rg * RPT + i) * kLd + d]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a[i][j] = fmaf(qx.w, kx[j].w, a[i][j]);
            a[i][j] = fmaf(qx.z, kx[j].z, a[i][j]);
            a[i][j] = fmaf(qx.y, kx[j].y, a[i][j]);
            a[i][j] = fmaf(qx.x, kx[j].x, a[i][j]);
          }
        }
      }
      const bool masked = key0 + kTile - 1 > low || key0 + kTile > s.limit;
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        float top = kNegInf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + cg + 16 * j;
          if (masked && (key >= s.limit || (pos[i] >= 0 && key > pos[i]))) a[i][j] = kNegInf;
          top = fmaxf(top, a[i][j]);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float next = fmaxf(m[i], top * p.scale_log2), ref = finite_or_zero(next);
        const float scale = ex2(m[i] - ref);
        m[i] = next;
        l[i] *= scale;
#pragma unroll
        for (int c = 0; c < 4 * kCols; ++c) o[i][c] *= scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[i][j] = ex2(fmaf(a[i][j], p.scale_log2, -ref));
          l[i] += a[i][j];
        }
      }
      __syncthreads();   // the keys have been read
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) weights[(rg * RPT + i) * kLdW + cg + 16 * j] = a[i][j];
      __syncwarp();      // a warp's rows are its own: no other warp reads them
#pragma unroll 2
      for (int key = 0; key < kTile; key += 4) {
        float4 vx[4][kCols];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            vx[t][c] = *reinterpret_cast<const float4*>(&sm.v[(key + t) * D + c * 64 + cg * 4]);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float4 w = *reinterpret_cast<const float4*>(&weights[(rg * RPT + i) * kLdW + key]);
          const float wt[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              o[i][4 * c] = fmaf(wt[t], vx[t][c].x, o[i][4 * c]);
              o[i][4 * c + 1] = fmaf(wt[t], vx[t][c].y, o[i][4 * c + 1]);
              o[i][4 * c + 2] = fmaf(wt[t], vx[t][c].z, o[i][4 * c + 2]);
              o[i][4 * c + 3] = fmaf(wt[t], vx[t][c].w, o[i][4 * c + 3]);
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = rg * RPT + i;
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
      if (r >= rows) continue;
      const bool real = pos[i] >= 0;   // padding rows are zero and weigh nothing
      const float sum = real ? l[i] : 0.f;
      const float f = !real ? 0.f : s.slot >= 0 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      const int64_t part = static_cast<int64_t>(s.slot) * p.row_tile + r;
      float* dst = s.slot < 0 ? static_cast<float*>(p.out) + query_row(r) : p.part_o + part * D;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        *reinterpret_cast<float4*>(dst + c * 64 + cg * 4) =
            real ? make_float4(o[i][4 * c] * f, o[i][4 * c + 1] * f, o[i][4 * c + 2] * f, o[i][4 * c + 3] * f)
                 : make_float4(0.f, 0.f, 0.f, 0.f);
      if (s.slot >= 0 && cg == 0)
        *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(real ? m[i] : kNegInf, sum);
    }
  }
}

template <int D, int RPT>
void launch(Args& args, int sms, cudaStream_t stream) {
  set_rows(args, 8 * RPT, kTile);
  const Split split(args, sms * kCtas<D, RPT>, 0, kItemCost);
  const size_t smem = sizeof(TileSmem<D, RPT>);
  auto kernel = paged_tile_fp32_kernel<D, RPT>;
  allow_smem(reinterpret_cast<const void*>(kernel), smem);
  kernel<<<split.ctas, kThreads, smem, stream>>>(args);
  EB_CUDA_CHECK(cudaGetLastError());
  count_launch(1);
  split.combine<float>(args, stream);
}

}  // namespace

void paged_tile_fp32_launch(Args& args, int sms, cudaStream_t stream) {
  // The smallest tile that takes all rows of a key head, or 64 rows. Four sequences over 30,000 keys,
  // 16 heads of 64, in tiles of 16 / 32 / 64 rows: 16 tokens 367 / 487 / 809 us, 32 tokens - / 487 / 809.
  const int64_t rows = static_cast<int64_t>(args.heads / args.kv_heads) * args.tokens;
  if (args.dim == 64) {
    if (rows <= 16) return launch<64, 2>(args, sms, stream);
    if (rows <= 32) return launch<64, 4>(args, sms, stream);
    return launch<64, 8>(args, sms, stream);
  }
  if (rows <= 16) return launch<128, 2>(args, sms, stream);
  if (rows <= 32) return launch<128, 4>(args, sms, stream);
  return launch<128, 8>(args, sms, stream);
}

}  // namespace eb
