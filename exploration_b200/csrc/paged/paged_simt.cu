// Attention of new tokens over a paged cache on the CUDA cores: fp32 inputs
// (IEEE fp32 products, no TF32) and head dims without a tensor-core form.
//
// out[r] = sum_{i <= pos_r} softmax(q_r . k_i / sqrt(D)) v_i, one pass over the
// keys with a running maximum and sum (base 2, fp32).
//
// One CTA of four warps walks its run of (item, key tile) pairs; a tile has 64
// keys, 16 a warp. Pages hold a power of two of at least 16 tokens, so a warp's
// 16 keys lie in one page and cost one table lookup, made one tile ahead. A key
// is spread over DP / 4 lanes (at most 32), four or eight elements each, read
// with 16-byte loads straight into registers: nothing is shared between warps
// until the end of an item, and the bytes in flight come from the occupancy.
// Up to R rows share each load. Measured: one token of two sequences of 60,001
// keys, 16 heads of 64, fp32 (0.98 GB): 0.151 to 0.155 ms, 6.3 to 6.5 TB/s, 97 to
// 99% of the measured copy bandwidth.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <type_traits>

#include "paged_common.cuh"
#include "paged_launch.h"

namespace eb {
namespace {

using namespace paged;

constexpr int kWarps = 4;
constexpr int kItemCost = 2;   // of an item's start and end, in tiles
constexpr int kTile = 64;
constexpr int kWholeTiles = 16;   // items of up to 1,024 keys are not cut (as in the few-row kernel)
constexpr int kWarpKeys = kTile / kWarps;

template <typename T, int VE>
EB_DEVICE void load_vec(const T* p, bool vec, int valid, float (&x)[VE]) {
  if (vec && valid >= VE) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(p + i);
        x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        const uint2 u = *reinterpret_cast<const uint2*>(p + i);
        const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int t = 0; t < 4; ++t) x[i + t] = load_f<T>(h + t);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = i < valid ? load_f<T>(p + i) : 0.f;
  }
}

template <typename T, int DP, int R>
__global__ void __launch_bounds__(kWarps * 32)
paged_simt_kernel(Args p) {
  constexpr int LK = DP / 4 < 32 ? DP / 4 : 32;   // lanes of a key
  constexpr int VE = DP / LK;
  constexpr int NG = 32 / LK;                     // keys side by side in a warp
  constexpr int U = DP == 256 ? 4 : (DP == 32 ? 4 : 8);
  constexpr int kPass = NG * U;
  using Sum = std::conditional_t<sizeof(T) == 4, double, float>;
  __shared__ Prefix table;
  __shared__ float sm_ml[kWarps][R][2];
  __shared__ float sm_o[kWarps][R][DP];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = lane / LK, d0 = (lane % LK) * VE;
  const int valid = p.dim - d0;                   // elements of this lane's vector that exist
  const bool vec = p.vectors != 0;
  if (p.flat) build_prefix(p, table);
  Walk walk;
  walk.start(p, table);
  publish_run<T>(p, table, walk);
  Segment s;
  const T* q = static_cast<const T*>(p.q);
  const T* kc = static_cast<const T*>(p.k);
  const T* vc = static_cast<const T*>(p.v);
  while (walk.next(p, table, s)) {
    finish_segment(p, table, s, lane);
    const int rows = min(p.tile_tokens, p.tokens - s.token0) * p.group;
    const int64_t row_base = static_cast<int64_t>(s.batch) * p.tokens + s.token0;
    float qr[R][VE], o[R][VE], m[R], l[R];
    int pos[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int rr = r < rows ? r : 0;
      const int64_t token = row_base + rr / p.group;
      pos[r] = r < rows ? p.positions[token] : -1;
      load_vec<T, VE>(q + (token * p.heads + s.head * p.group + rr % p.group) * p.dim + d0, vec, valid, qr[r]);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        qr[r][i] *= p.scale_log2;
        o[r][i] = 0.f;
      }
      m[r] = kNegInf;
      l[r] = 0.f;
    }
    const int* pages = p.tables + static_cast<int64_t>(s.batch) * p.width;
    const int64_t head_step = static_cast<int64_t>(p.page) * p.dim;
    const int kv_head = s.head / p.head_div;
    auto page_of = [&](int tile) {
      const int key = tile * kTile + warp * kWarpKeys;
      return tile < s.end && key < s.limit ? pages[key >> p.page_shift] : -1;
    };
    int next_id = page_of(s.begin);
    for (int tile = s.begin; tile < s.end; ++tile) {
      const int id = next_id;
      next_id = page_of(tile + 1);
      if (id < 0 || id >= p.pages) continue;
      const int64_t base = (static_cast<int64_t>(id) * p.kv_heads + kv_head) * head_step;
#pragma unroll 1
      for (int pass = 0; pass < kWarpKeys; pass += kPass) {
        const int key0 = tile * kTile + warp * kWarpKeys + pass + grp;
        float kx[U][VE], vx[U][VE];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int key = key0 + u * NG;
          const int64_t at = base + static_cast<int64_t>(key & (p.page - 1)) * p.dim + d0;
          const int n = key < s.limit ? valid : 0;
          load_vec<T, VE>(kc + at, vec, n, kx[u]);
          load_vec<T, VE>(vc + at, vec, n, vx[u]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r >= rows) break;
          float a[U];
          float top = kNegInf;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float dot = 0.f;
#pragma unroll
            for (int i = VE - 1; i >= 0; --i) dot = fmaf(qr[r][i], kx[u][i], dot);
            // fp32 inputs: the lanes' parts are added in fp64, so a logit of size 2^9 is off by two roundings, not five.
            Sum total = dot;
#pragma unroll
            for (int off = LK / 2; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
            a[u] = key0 + u * NG <= pos[r] ? static_cast<float>(total) : kNegInf;
            top = fmaxf(top, a[u]);
          }
#pragma unroll
          for (int off = LK; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float next = fmaxf(m[r], top), ref = finite_or_zero(next);
          const float scale = ex2(m[r] - ref);
          m[r] = next;
          l[r] *= scale;
#pragma unroll
          for (int i = 0; i < VE; ++i) o[r][i] *= scale;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bool seen = key0 + u * NG <= pos[r];
            const float w = ex2(a[u] - ref);
            l[r] += w;
            if (seen) {   // a value that this row does not see may be anything, NaN included
#pragma unroll
              for (int i = 0; i < VE; ++i) o[r][i] = fmaf(w, vx[u][i], o[r][i]);
            }
          }
        }
      }
    }
    // Lane groups, then warps.
    __syncthreads();   // the previous item's sums have been read
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int off = LK; off < 32; off <<= 1) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
#pragma unroll
        for (int i = 0; i < VE; ++i) o[r][i] += __shfl_xor_sync(0xffffffffu, o[r][i], off);
      }
      if (lane == 0) {
        sm_ml[warp][r][0] = m[r];
        sm_ml[warp][r][1] = l[r];
      }
      if (grp == 0) {
#pragma unroll
        for (int i = 0; i < VE; ++i) sm_o[warp][r][d0 + i] = o[r][i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * DP; i += blockDim.x) {
      const int r = i / DP, d = i % DP;
      if (d >= p.dim) continue;
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_ml[w][r][0]);
      const float ref = finite_or_zero(top);
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sm_ml[w][r][0] - ref);
        sum += f * sm_ml[w][r][1];
        acc += f * sm_o[w][r][d];
      }
      if (s.slot < 0) {
        const int64_t token = row_base + r / p.group;
        static_cast<T*>(p.out)[(token * p.heads + s.head * p.group + r % p.group) * p.dim + d] =
            cast_f<T>(sum == 0.f ? 0.f : acc / sum);
      } else {
        const int64_t row = static_cast<int64_t>(s.slot) * p.row_tile + r;
        p.part_o[row * p.dim + d] = acc;
        if (d == 0) {
          p.part_ml[row * 2] = top;
          p.part_ml[row * 2 + 1] = sum;
        }
      }
    }
  }
}

template <typename T, int DP, int R>
void launch(Args& args, int sms, cudaStream_t stream) {
  const Split split(args, sms * 4, kWholeTiles, kItemCost);
  paged_simt_kernel<T, DP, R><<<split.ctas, kWarps * 32, 0, stream>>>(args);
  EB_CUDA_CHECK(cudaGetLastError());
  count_launch(1);
  split.combine<T>(args, stream);
}

template <typename T, int R>
void by_dim(Args& args, int sms, cudaStream_t stream) {
  if (args.dim <= 32) return launch<T, 32, R>(args, sms, stream);
  if (args.dim <= 64) return launch<T, 64, R>(args, sms, stream);
  if (args.dim <= 128) return launch<T, 128, R>(args, sms, stream);
  return launch<T, 256, R>(args, sms, stream);
}

}  // namespace

template <typename T>
void paged_simt_launch(Args& args, int sms, cudaStream_t stream) {
  const int group = args.heads / args.kv_heads;
  // Rows that share a load: one for single tokens without shared heads (one token of four sequences over
  // 30,000 keys, 16 heads of 64, fp32: 157 us, 182 us in the form for eight), else up to eight.
  const int most = static_cast<int64_t>(group) * args.tokens == 1 ? 1 : 8;
  set_rows(args, most, kTile);
  if (most == 1) return by_dim<T, 1>(args, sms, stream);
  return by_dim<T, 8>(args, sms, stream);
}

template void paged_simt_launch<float>(Args&, int, cudaStream_t);
template void paged_simt_launch<__half>(Args&, int, cudaStream_t);
template void paged_simt_launch<__nv_bfloat16>(Args&, int, cudaStream_t);

}  // namespace eb
