// Attention of few rows over a paged cache (16-bit types, head dim 64 or 128):
// up to 16 rows of one (sequence, key head), i.e. single tokens, a few drafted
// tokens, the query heads that share a key head.
//
// Bound by one read of the keys and values. A producer warp streams 64-key
// tiles with TMA (one box a page, 128-byte swizzle) through a ring of stages;
// four consumer warps take 16 keys of each tile and never wait for each other
// inside an item: each keeps a running maximum, sum and accumulator for all 16
// rows, joined through shared memory at the item's end. With at most 16 rows a
// tile needs 0.5 MFLOP per 16 KB (head dim 64), far below what the warp-level
// m16n8k16 instruction gives, and its fragments come from registers without the
// round trip through tensor memory (and without padding 16 rows to 128) that
// tcgen05 would cost here; arithmetic hides under the loads.
//
// Measured: one token of 64 sequences of 17 to 16,384 keys, 32/8 heads of 128,
// bf16 (2.15 GB): 0.330 to 0.344 ms, 6.3 to 6.5 TB/s, 95 to 99% of the measured copy
// bandwidth. Five tokens of 16 sequences of up to 4,099 keys, 16 heads of 64, fp16
// (148 MB): 30 us of kernel, bound by its start (positions, tables, first tiles:
// 4 us) and by the joining launch after it (5 us).
//
// Keys past an item's limit are masked, their values cleared in the fragments:
// a page's unwritten rows may hold anything.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <climits>

#include "../common/sm100.cuh"
#include "../common/tma.cuh"
#include "paged_common.cuh"
#include "paged_launch.h"
#include "paged_mma.cuh"

namespace eb {
namespace {

using namespace paged;
using namespace sm100;

constexpr int kRows = 16;
constexpr int kItemCost = 2;   // of an item's start and end, in tiles
constexpr int kTile = 64;
// Items of up to 1,024 keys are not cut, because joining costs a launch: 4 sequences of
// up to 517 keys, 4 heads of 64, take one kernel of 8.1 us whole, 5.3 + 3.5 us cut.
constexpr int kWholeTiles = 16;
constexpr int kConsumers = 4;
constexpr int kThreads = 32 * (kConsumers + 1);

// CTAs an SM and stages of each, within shared memory and registers (head dim 64: three
// CTAs of three stages 38.1 us for the drafted tokens above, two of five 39.0 us).
template <int D>
struct RowsConfig;
template <>
struct RowsConfig<64> {
  static constexpr int kStages = 3, kCtas = 3;
};
template <>
struct RowsConfig<128> {
  static constexpr int kStages = 5, kCtas = 1;
};

template <int D>
struct alignas(1024) RowsSmem {
  static constexpr int kStages = RowsConfig<D>::kStages;
  uint16_t kv[kStages][2][kTile * D];       // [keys, values][d / 64][key][64], swizzled
  float o[kConsumers][kRows][D];
  float ml[kConsumers][kRows][2];
  uint64_t full[kStages], empty[kStages];
  int abort;
  Prefix table;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, RowsConfig<D>::kCtas)
paged_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, Args p,
                  ErrorSlot* err) {
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  RowsSmem<D>& sm = *reinterpret_cast<RowsSmem<D>*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr int kStages = RowsSmem<D>::kStages;
  constexpr int kHalf = kTile * 64;              // elements of a 64-wide half
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], kConsumers);
    }
    sm.abort = 0;
    fence_barrier_init();
  }
  if (p.flat) build_prefix(p, sm.table);
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Walk walk;
  walk.start(p, sm.table);
  publish_run<T>(p, sm.table, walk);
  Segment s;

  if (warp == kConsumers) {
    // Producer. Table entries are read 32 pages at a time, one group ahead.
    const int box = min(p.page, kTile);
    const int pages_tile = kTile / box;
    if (lane == 0) {
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
    }
    int issued = 0;
    bool ok = true;
    while (ok && walk.next(p, sm.table, s)) {
      // The first entries are on their way before the limit is known (the table has them all).
      const int* table = p.tables + static_cast<int64_t>(s.batch) * p.width;
      const int kv_head = s.head / p.head_div;
      auto entry = [&](int page) { return page < p.width ? table[page] : -1; };
      int base = p.flat ? (s.begin * kTile) >> p.page_shift : 0;
      int ids = entry(base + lane), ahead = entry(base + 32 + lane);
      finish_segment(p, sm.table, s, lane);
      for (int tile = s.begin; tile < s.end; ++tile) {
        const int stage = issued % kStages;
        if (issued >= kStages && !__all_sync(0xffffffffu, wait_tight(&sm.empty[stage], ((issued / kStages) - 1) & 1,
                                                                    abort, err, kSiteKvEmpty))) {
          ok = false;
          break;
        }
        const int key0 = tile * kTile;
        const int boxes = min(pages_tile, cdiv(s.limit - key0, box));
        // Lane i fetches box i (at most four a tile). An entry outside the pool reads as
        // zeros (out of the map's bounds), never foreign memory.
        if ((key0 >> p.page_shift) - base >= 32) {
          base += 32;
          ids = ahead;
          ahead = entry(base + 32 + lane);
        }
        const int want = ((key0 + min(lane, boxes - 1) * box) >> p.page_shift) - base;
        const int id_low = __shfl_sync(0xffffffffu, ids, want & 31), id_high = __shfl_sync(0xffffffffu, ahead, want & 31);
        const int id = want < 32 ? id_low : id_high;
        const int plane = id >= 0 && id < p.pages ? id * p.kv_heads + kv_head : p.pages * p.kv_heads;
        if (lane == 0) mbar_expect_tx(&sm.full[stage], boxes * box * D * 2 * 2);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            tma_load_3d(&sm.kv[stage][0][h * kHalf + lane * box * 64], &tk, &sm.full[stage], h * 64,
                        (key0 + lane * box) & (p.page - 1), plane);
            tma_load_3d(&sm.kv[stage][1][h * kHalf + lane * box * 64], &tv, &sm.full[stage], h * 64,
                        (key0 + lane * box) & (p.page - 1), plane);
          }
        }
        ++issued;
      }
    }
    if (*abort && lane == 0) {   // let issued copies land before the CTA exits
      for (int j = max(0, issued - kStages); j < issued; ++j)
        mbar_wait(&sm.full[j % kStages], (j / kStages) & 1, abort, nullptr, kSiteDrain);
    }
    return;
  }

  const T* q = static_cast<const T*>(p.q);
  int done = 0;
  bool ok = true;
  while (ok && walk.next(p, sm.table, s)) {
    const int rows = min(p.tile_tokens, p.tokens - s.token0) * p.group;
    const int64_t row_base = static_cast<int64_t>(s.batch) * p.tokens + s.token0;
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    // Rows r0 and r0 + 8 of this thread: position and query fragments.
    int pos[2];
    uint32_t qa[D / 16][4];
    int top = -1, low = INT_MAX;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + 8 * i, rr = r < rows ? r : 0;
      const int64_t token = row_base + rr / p.group;
      pos[i] = r < rows ? p.positions[token] : -1;
      const T* src = q + (token * p.heads + s.head * p.group + rr % p.group) * D + c0;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qa[k][i] = *reinterpret_cast<const uint32_t*>(src + k * 16);
        qa[k][2 + i] = *reinterpret_cast<const uint32_t*>(src + k * 16 + 8);
      }
      top = max(top, pos[i]);
      if (pos[i] >= 0) low = min(low, pos[i]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    s.limit = static_cast<int>(min(static_cast<int64_t>(top) + 1, static_cast<int64_t>(p.width) * p.page));
    if (!p.flat) {
      s.begin = 0;
      s.end = cdiv(s.limit, kTile);
    }
    // Absent rows see everything (their zeros or copies are never written), so that
    // only tiles with the last keys of some row need a mask.
    const int see0 = pos[0] >= 0 ? pos[0] : INT_MAX, see1 = pos[1] >= 0 ? pos[1] : INT_MAX;
    float m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    for (int tile = s.begin; tile < s.end; ++tile, ++done) {
      const int stage = done % kStages;
      if (!__all_sync(0xffffffffu, wait_tight(&sm.full[stage], (done / kStages) & 1, abort, err, kSiteKvFull))) {
        ok = false;
        break;
      }
      const int key0 = tile * kTile + warp * 16;
      if (key0 < s.limit) {
        const uint32_t k_base = smem_u32(&sm.kv[stage][0][0]) + warp * 16 * 128;
        const uint32_t v_base = smem_u32(&sm.kv[stage][1][0]) + warp * 16 * 128;
        float a[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[0][i] = a[1][i] = 0.f;
        {
          const int row = (lane & 7) + ((lane >> 4) << 3), part = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            const int chunk = (2 * k + part) & 7;
            ldmatrix4(b, k_base + (k / 4) * kHalf * 2 + row * 128 + ((chunk ^ (row & 7)) << 4));
            mma16816<T>(a[0], qa[k], b[0], b[1]);
            mma16816<T>(a[1], qa[k], b[2], b[3]);
          }
        }
        if (key0 + 15 > low || key0 + 16 > s.limit) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int key = key0 + n * 8 + c0 + i;
              if (key > see0 || key >= s.limit) a[n][i] = kNegInf;
              if (key > see1 || key >= s.limit) a[n][2 + i] = kNegInf;
            }
        }
        float scale[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float t = fmaxf(fmaxf(a[0][2 * i], a[0][2 * i + 1]), fmaxf(a[1][2 * i], a[1][2 * i + 1]));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
          const float next = fmaxf(m[i], reference_point(t, p.scale_log2, kWeightExp<T>)), ref = finite_or_zero(next);
          scale[i] = ex2(m[i] - ref);
          m[i] = next;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float w = ex2(fmaf(a[n][2 * i + j], p.scale_log2, -ref));
              a[n][2 * i + j] = w;
              sum += w;
            }
          l[i] = l[i] * scale[i] + sum;
        }
        if (__any_sync(0xffffffffu, scale[0] != 1.f || scale[1] != 1.f)) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][0] *= scale[0];
            o[n][1] *= scale[0];
            o[n][2] *= scale[1];
            o[n][3] *= scale[1];
          }
        }
        // Weights are rounded to the input type for the second product (their sum is not): at most
        // 2^15 in fp16, so that keys 2^-29 below the largest keep their bits.
        const uint32_t w[4] = {pack2<T>(a[0][0], a[0][1]), pack2<T>(a[0][2], a[0][3]), pack2<T>(a[1][0], a[1][1]),
                               pack2<T>(a[1][2], a[1][3])};
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        const bool ragged = key0 + 16 > s.limit;
        if (ragged) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
            keep[n] = (key0 + n * 8 + c0 < s.limit ? 0xffffu : 0u) |
                      (key0 + n * 8 + c0 + 1 < s.limit ? 0xffff0000u : 0u);
        }
        {
          const int row = (lane & 7) + (((lane >> 3) & 1) << 3), part = lane >> 4;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t b[4];
            const int chunk = (2 * c + part) & 7;
            ldmatrix4_trans(b, v_base + (c / 4) * kHalf * 2 + row * 128 + ((chunk ^ (row & 7)) << 4));
            if (ragged) {
              b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
            }
            mma16816<T>(o[2 * c], w, b[0], b[1]);
            mma16816<T>(o[2 * c + 1], w, b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[stage]);
    }
    if (!ok) break;
    // Sums of the quad's columns, then the four warps through shared memory.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      const int r = r0 + 8 * i;
      if (r < rows) {
        const bool real = pos[i] >= 0;
        if ((lane & 3) == 0) {
          sm.ml[warp][r][0] = real ? m[i] : kNegInf;
          sm.ml[warp][r][1] = real ? l[i] : 0.f;
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(&sm.o[warp][r][n * 8 + c0]) =
              real ? make_float2(o[n][2 * i], o[n][2 * i + 1]) : make_float2(0.f, 0.f);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");
    for (int i = threadIdx.x; i < rows * (D / 2); i += 32 * kConsumers) {
      const int r = i / (D / 2), d = (i % (D / 2)) * 2;
      float best = kNegInf;
#pragma unroll
      for (int c = 0; c < kConsumers; ++c) best = fmaxf(best, sm.ml[c][r][0]);
      const float ref = finite_or_zero(best);
      float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int c = 0; c < kConsumers; ++c) {
        const float f = ex2(sm.ml[c][r][0] - ref);
        const float2 part = *reinterpret_cast<const float2*>(&sm.o[c][r][d]);
        sum += f * sm.ml[c][r][1];
        x += f * part.x;
        y += f * part.y;
      }
      if (s.slot < 0) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t token = row_base + r / p.group;
        *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) +
                                     (token * p.heads + s.head * p.group + r % p.group) * D + d) =
            pack2<T>(x * inv, y * inv);
      } else {
        const int64_t row = static_cast<int64_t>(s.slot) * p.row_tile + r;
        *reinterpret_cast<float2*>(p.part_o + row * D + d) = make_float2(x, y);
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + row * 2) = make_float2(best, sum);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");
  }
}

template <typename T, int D>
void launch(Args& args, int sms, cudaStream_t stream) {
  const Split split(args, sms * RowsConfig<D>::kCtas, kWholeTiles, kItemCost);
  const CUtensorMap tk = make_pool_map(args, args.k, std::is_same_v<T, __half>, kTile);
  const CUtensorMap tv = make_pool_map(args, args.v, std::is_same_v<T, __half>, kTile);
  const size_t smem = sizeof(RowsSmem<D>) + 1024;
  auto kernel = paged_rows_kernel<T, D>;
  allow_smem(reinterpret_cast<const void*>(kernel), smem);
  kernel<<<split.ctas, kThreads, smem, stream>>>(tk, tv, args, device_error_slot(at::cuda::current_device()));
  EB_CUDA_CHECK(cudaGetLastError());
  count_launch(1);
  split.combine<T>(args, stream);
}

}  // namespace

template <typename T>
void paged_rows_launch(Args& args, int sms, cudaStream_t stream) {
  set_rows(args, kRows, kTile);
  if (args.dim == 64) return launch<T, 64>(args, sms, stream);
  return launch<T, 128>(args, sms, stream);
}

template void paged_rows_launch<__half>(Args&, int, cudaStream_t);
template void paged_rows_launch<__nv_bfloat16>(Args&, int, cudaStream_t);

}  // namespace eb
