// Attention of a chunk of new tokens over a paged cache on the 5th-generation
// tensor cores (16-bit types, head dim 64 or 128, more than 16 rows of a key head).
//
// out[r] = sum_{i <= pos_r} softmax(q_r . k_i / sqrt(D)) v_i with the running
// maximum and sum of one pass (base 2, fp32). Rows are packed token by token,
// the query heads of a key head side by side, so small chunks with shared heads
// still fill the 128 rows of an MMA.
//
// One CTA walks its run of (item, 128-key tile) pairs. Warp roles (384 threads):
//   warp 0       producer: Q once an item, K and V tiles (a TMA box a page,
//                128-byte swizzle) into two rings
//   warp 1       MMA issuer: S = Q K^T into TMEM, O += P V with P read from TMEM
//   warp 2       TMEM owner (512 columns)
//   warp 3       clears the rows past an item's limit in its last V tile
//   warps 4-7    softmax warpgroup 0, one thread a row (TMEM lane)
//   warps 8-11   softmax warpgroup 1
// Items of more than 128 rows give each warpgroup its own 128 rows of every key
// tile; smaller ones give both the same rows and alternate key tiles, joined
// through TMEM at the item's end. Either way the issuer alternates between the
// warpgroups: while one exponentiates its scores, the other's products run.
//
// P (16 bit) overwrites its scores' TMEM columns; steps use the score buffers in
// turn (three at head dim 64, two at 128), so with three a warpgroup finds its
// next scores ready. A row's reference point is kept until its maximum has grown past
// it by more than 2^8 (2^4 in fp16); then O is rescaled in TMEM.
//
// TMEM columns: score buffers from 0, then the two accumulators of D columns.
//
// Measured: 2,048 tokens over 65,536 keys, 16 heads of 64, bf16: 0.64 ms in a short
// burst (850 TFLOP/s), 0.76 ms sustained under the power cap (713); ragged chunks of
// 1,111 tokens over up to 8,191 keys, 32/8 heads of 128, fp16: 0.37 and 0.43 ms (780).
// At head dim 64 a step is bound by the softmax instructions of two warps an SM
// sub-partition (their special-function share alone is 2,048 cycles of 2,500) and the
// hand-overs around them; at 128 by the chain weights -> P V -> next S -> softmax
// (3,300 cycles for 2,056 of tensor work). A finished barrier costs a waiting warp some
// 90 cycles, so what did not pay: exponentials on the FMA pipe, two issuing threads,
// scores released early, strict turns of the warpgroups, shorter steps.
//
// Non-finite values of a key that some row of the call sees may reach its other
// rows: a weight of zero times a NaN is a NaN in the matrix unit.
//
// Keys past an item's limit are masked, and their V rows cleared: a page's
// unwritten rows may hold anything.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <climits>

#include "../common/sm100.cuh"
#include "../common/tma.cuh"
#include "paged_common.cuh"
#include "paged_launch.h"
#include "paged_mma.cuh"
#include "paged_phases.h"

namespace eb {
namespace {

using namespace paged;
using namespace sm100;

constexpr int kM = 128;               // rows of an MMA
constexpr int kItemCost = 3;   // of an item's start and end, in tiles
constexpr int kTile = 128;            // keys of a tile
constexpr int kBox = 128 * 64;        // elements of a 64-wide half of a 128-row operand
constexpr int kThreads = 384;
constexpr int kTmemCols = 512;
// How far a row's maximum may grow past its reference point before the accumulator is rescaled
// (log2 units). In fp16 every unit of it is taken from the range of the weights (paged_mma.cuh): with 4
// keys 2^-25 below the largest keep all bits, with 8 2^-21. Logits of standard deviation 2, ragged chunks
// of 1,111 tokens over up to 8,191 keys, in a burst: 351 us with 8, 367 with 4, 385 with 2; 2,048
// tokens over 32,768 keys, head dim 64: 328 us with 8, 347 with 4.
template <typename T>
constexpr float kRescale = std::is_same_v<T, __half> ? 4.f : 8.f;

template <int D>
struct alignas(1024) ChunkSmem {
  static constexpr int kStages = D == 64 ? 4 : 2;   // of each ring
  static constexpr int kBufs = (kTmemCols - 2 * D) / 128;   // score buffers in TMEM
  // With two buffers the next scores wait for this step's products: those of the
  // first half of the keys begin while the second half's weights are computed.
  static constexpr bool kHalves = kBufs == 2;
  uint16_t q[2][kM * D];
  uint16_t k[kStages][kTile * D];
  uint16_t v[kStages][kTile * D];
  uint64_t q_full, q_empty;
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[kBufs], p_full[kBufs], p_half[kBufs], join, v_ragged, v_clear, drained;
  uint64_t o_done[2][kProductBarriers];   // of each warpgroup, its products in turn (paged_phases.h)
  uint32_t tmem_base;
  int abort;
  int clear_stage;
  float ml[kM][2];
  Prefix table;
};

// Positions in the two rings and of the barriers' phases, carried across items.
struct Ring {
  int stage = 0, phase = 0;
  EB_DEVICE void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// Keeps the compiler from using TMEM loads before the wait that precedes this.
template <int N>
EB_DEVICE void hold(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// True in one lane of a converged warp; unlike a comparison of lane numbers it
// lets the compiler keep the operands of the guarded instructions uniform.
EB_DEVICE bool elect_one() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred != 0;
}

// Shared-memory matrix descriptors (128-byte swizzle, 1,024 bytes between groups of
// eight rows) in two words: only the low one, address and leading offset, changes.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);

EB_DEVICE uint32_t desc_lo(const void* ptr, uint32_t leading_bytes) {
  return (smem_u32(ptr) >> 4) | ((leading_bytes >> 4) << 16);
}

template <uint32_t HI>
EB_DEVICE void mma_ss_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(HI)
      : "memory");
}

template <uint32_t HI>
EB_DEVICE void mma_ts_lo(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(HI)
      : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, Args p, ErrorSlot* err) {
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  ChunkSmem<D>& sm = *reinterpret_cast<ChunkSmem<D>*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr int kStages = ChunkSmem<D>::kStages, kBufs = ChunkSmem<D>::kBufs;
  constexpr bool kHalves = ChunkSmem<D>::kHalves;
  constexpr int kO = kTmemCols - 2 * D;          // first TMEM column of the accumulators
  static_assert(kProductBarriers == 2, "the issuer keeps each warpgroup's turn in one bit");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sm.abort;
  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&sm.s_full[b], 1);
      mbar_init(&sm.p_full[b], 128);
      mbar_init(&sm.p_half[b], 128);
    }
    for (int w = 0; w < 2; ++w)
      for (uint32_t b = 0; b < kProductBarriers; ++b) mbar_init(&sm.o_done[w][b], 1);
    mbar_init(&sm.join, 256);
    mbar_init(&sm.v_ragged, 1);
    mbar_init(&sm.v_clear, 1);
    mbar_init(&sm.drained, 1);
    sm.abort = 0;
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc(&sm.tmem_base, kTmemCols);
  if (p.flat) build_prefix(p, sm.table);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;
  Walk walk;
  walk.start(p, sm.table);
  publish_run<T>(p, sm.table, walk);
  Segment s;
  const int half_tokens = kM / p.group;         // tokens of one warpgroup's rows
  const int half_rows = half_tokens * p.group;
  // Both warpgroups have rows of their own when the item holds more tokens than one takes.
  auto split_rows = [&](const Segment& seg) { return p.tokens - seg.token0 > half_tokens; };

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 0) {
    const int box = min(p.page, kTile), boxes_tile = kTile / box;
    if (lane == 0) {
      prefetch_tensormap(&tq);
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
    }
    CopyRing k_ring, v_ring;
    int q_loads = 0;
    bool ok = true;
    while (ok && walk.next(p, sm.table, s)) {
      // The first entries are on their way before the limit is known (the table has them all).
      const int* table = p.tables + static_cast<int64_t>(s.batch) * p.width;
      const int kv_head = s.head / p.head_div;
      auto entry = [&](int page) { return page < p.width ? table[page] : -1; };
      int base = p.flat ? (s.begin * kTile) >> p.page_shift : 0;
      int ids = entry(base + lane), ahead = entry(base + 32 + lane);
      finish_segment(p, sm.table, s, lane);
      if (s.begin == s.end) continue;
      if (q_loads > 0 && !__all_sync(0xffffffffu, wait_tight(&sm.q_empty, (q_loads - 1) & 1, abort, err, kSiteQFull)))
        break;
      const int halves = split_rows(s) ? 2 : 1;
      if (lane == 0) {
        mbar_expect_tx(&sm.q_full, halves * half_rows * D * 2);
        for (int w = 0; w < halves; ++w)
#pragma unroll
          for (int h = 0; h < D / 64; ++h)
            tma_load_4d(&sm.q[w][h * kBox], &tq, &sm.q_full, h * 64, s.head * p.group, s.token0 + w * half_tokens,
                        s.batch);
      }
      ++q_loads;
      for (int tile = s.begin; tile < s.end; ++tile) {
        const int key0 = tile * kTile;
        const int boxes = min(boxes_tile, cdiv(s.limit - key0, box));
        // Plane of box i in lane i (at most eight boxes a tile). An entry outside
        // the pool reads as zeros (out of the map's bounds), never foreign memory.
        const int first_page = key0 >> p.page_shift;
        if (first_page - base >= 32) {
          base += 32;
          ids = ahead;
          ahead = entry(base + 32 + lane);
        }
        const int want = ((key0 + min(lane, boxes - 1) * box) >> p.page_shift) - base;
        const int id_low = __shfl_sync(0xffffffffu, ids, want & 31), id_high = __shfl_sync(0xffffffffu, ahead, want & 31);
        const int id = want < 32 ? id_low : id_high;
        const int plane = id >= 0 && id < p.pages ? id * p.kv_heads + kv_head : p.pages * p.kv_heads;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          CopyRing& ring = part == 0 ? k_ring : v_ring;
          const Phase slot = ring.next(kStages);
          uint64_t* full = part == 0 ? &sm.k_full[slot.barrier] : &sm.v_full[slot.barrier];
          uint64_t* empty = part == 0 ? &sm.k_empty[slot.barrier] : &sm.v_empty[slot.barrier];
          uint16_t* dst = part == 0 ? sm.k[slot.barrier] : sm.v[slot.barrier];
          const CUtensorMap* map = part == 0 ? &tk : &tv;
          if (ring.reuses(kStages) &&
              !__all_sync(0xffffffffu, wait_tight(empty, slot.parity ^ 1, abort, err, kSiteKvEmpty))) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(full, boxes * box * D * 2);
          __syncwarp();
          if (lane < boxes) {
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
              tma_load_3d(dst + h * kBox + lane * box * 64, map, full, h * 64, (key0 + lane * box) & (p.page - 1),
                          plane);
          }
          ++ring.issued;
        }
        if (!ok) break;
      }
    }
    if (*abort && lane == 0) {   // let issued copies land before the CTA exits
      k_ring.drain(kStages, [&](uint32_t stage, uint32_t parity) {
        mbar_wait(&sm.k_full[stage], parity, abort, nullptr, kSiteDrain);
      });
      v_ring.drain(kStages, [&](uint32_t stage, uint32_t parity) {
        mbar_wait(&sm.v_full[stage], parity, abort, nullptr, kSiteDrain);
      });
      if (q_loads > 0) mbar_wait(&sm.q_full, (q_loads - 1) & 1, abort, nullptr, kSiteDrain);
    }
  } else if (warp == 1) {
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    const uint32_t id_s = idesc_16(kBf16, kM, kTile, false, false);
    const uint32_t id_pv = idesc_16(kBf16, kM, D, false, true);
    Ring kr, vr, sr, pr;    // key and value stages, score buffers to fill and weights to use
    int segments = 0, cleared = 0;
    uint32_t turn = 0;      // bit w: barrier of warpgroup w's next product (product_phase)
    bool ok = true;
    while (ok && walk.next(p, sm.table, s)) {
      finish_segment(p, sm.table, s, lane);
      if (s.begin == s.end) continue;
      const bool dual = split_rows(s);
      const int tiles = s.end - s.begin, steps = dual ? 2 * tiles : tiles;
      const int ragged = s.limit < s.end * kTile ? s.end - 1 : -1;   // tile whose values warp 3 clears
      const int q_phase = segments & 1, clear_phase = cleared & 1;
      ++segments;
      cleared += ragged >= 0;
      // One thread does all of an item: a warp-wide wait costs a vote, and there are three a step.
      if (elect_one()) {
        // Step i belongs to warpgroup i & 1; with rows of their own both take each tile.
        auto issue_s = [&](int i) {
          const int w = i & 1;
          if (!dual || w == 0) ok = ok && wait_tight(&sm.k_full[kr.stage], kr.phase, abort, err, kSiteKvFull);
          if (!ok) return;
          tc_fence_after();
          const uint32_t q_lo = desc_lo(sm.q[dual ? w : 0], 16), k_lo = desc_lo(sm.k[kr.stage], 16);
          const uint32_t d_addr = tmem + sr.stage * 128;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * kBox * 2 + (kk % 4) * 32;
            mma_ss_lo<kDescHi>(d_addr, q_lo + (off >> 4), k_lo + (off >> 4), id_s, kk > 0);
          }
          tc_commit(&sm.s_full[sr.stage]);
          if (i == steps - 1) tc_commit(&sm.q_empty);
          sr.next(kBufs);
          if (!dual || w == 1) {
            tc_commit(&sm.k_empty[kr.stage]);
            kr.next(kStages);
          }
        };
        ok = wait_tight(&sm.q_full, q_phase, abort, err, kSiteQFull);
        for (int i = 0; ok && i < min(kBufs, steps); ++i) issue_s(i);
        for (int i = 0; ok && i < steps; ++i) {
          const int w = i & 1, tile = s.begin + (dual ? i >> 1 : i);
          if (!dual || w == 0) {
            ok = wait_tight(&sm.v_full[vr.stage], vr.phase, abort, err, kSiteKvFull);
            if (ok && tile == ragged) {
              sm.clear_stage = vr.stage;
              mbar_arrive(&sm.v_ragged);
              ok = wait_tight(&sm.v_clear, clear_phase, abort, err, kSiteKvFull);
            }
          }
          ok = ok && wait_tight(kHalves ? &sm.p_half[pr.stage] : &sm.p_full[pr.stage], pr.phase, abort, err, kSitePFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t v_lo = desc_lo(sm.v[vr.stage], kBox * 2);
          const uint32_t o_addr = tmem + kO + w * D, p_addr = tmem + pr.stage * 128, more = i > 1;
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk) {
            if (kHalves && kk == kTile / 32) {
              ok = wait_tight(&sm.p_full[pr.stage], pr.phase, abort, err, kSitePFull);
              if (!ok) break;
              tc_fence_after();
            }
            mma_ts_lo<kDescHi>(o_addr, p_addr + kk * 8, v_lo + kk * (2048 >> 4), id_pv, kk > 0 ? 1u : more);
          }
          if (!ok) break;
          tc_commit(&sm.o_done[w][turn >> w & 1]);
          turn ^= 1u << w;
          pr.next(kBufs);
          if (!dual || w == 1) {
            tc_commit(&sm.v_empty[vr.stage]);
            vr.next(kStages);
          }
          if (i + kBufs < steps) issue_s(i + kBufs);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
    if (*abort && elect_one()) {   // issued products read shared memory and TMEM: let them end first
      tc_commit(&sm.drained);
      mbar_wait(&sm.drained, 0, abort, nullptr, kSiteDrain);
    }
  } else if (warp == 3) {
    // Rows past an item's limit in its last value tile: cleared when warp 1 has seen the tile arrive.
    int cleared = 0;
    bool ok = true;
    while (ok && walk.next(p, sm.table, s)) {
      finish_segment(p, sm.table, s, lane);
      if (s.begin == s.end || s.limit >= s.end * kTile) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(&sm.v_ragged, cleared & 1, abort, err, kSiteKvFull));
      if (!ok) break;
      ++cleared;
      const int stage = *static_cast<volatile int*>(&sm.clear_stage);
      uint4* rows = reinterpret_cast<uint4*>(sm.v[stage]);
      for (int j = (s.limit - (s.end - 1) * kTile) * 8 + lane; j < kTile * 8; j += 32)
#pragma unroll
        for (int h = 0; h < D / 64; ++h) rows[h * (kBox / 8) + j] = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.v_clear);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = (warp >> 2) - 1;                   // softmax warpgroup
    const int row = (warp & 3) * 32 + lane;          // TMEM lane
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t o_addr = lane_addr + kO + w * D;
    constexpr float kBelow = std::is_same_v<T, __half> ? kWeightExp<T> - kRescale<T> : 0.f;
    int joins = 0;
    uint32_t done = 0;       // products this warpgroup has asked for
    uint32_t step0 = 0;      // steps of earlier items, both warpgroups'
    bool ok = true;
    // The last product that this warpgroup asked for.
    auto product_done = [&]() -> bool {
      const Phase phase = product_phase(done - 1);
      return __all_sync(0xffffffffu, wait_tight(&sm.o_done[w][phase.barrier], phase.parity, abort, err, kSiteODone));
    };
    // Both warpgroups, bounded: TMEM accesses before it are ordered before those after it.
    auto join = [&]() -> bool {
      tc_fence_before();
      mbar_arrive(&sm.join);
      const bool met = __all_sync(0xffffffffu, wait_tight(&sm.join, joins & 1, abort, err, kSiteODone));
      ++joins;
      tc_fence_after();
      return met;
    };
    while (ok && walk.next(p, sm.table, s)) {
      finish_segment(p, sm.table, s, lane);
      const bool dual = split_rows(s);
      const int first = dual ? w * half_tokens : 0;
      const int token = s.token0 + first + row / p.group;
      const bool present = row < half_rows && token < p.tokens;
      const int64_t flat_token = static_cast<int64_t>(s.batch) * p.tokens + token;
      const int pos = present ? p.positions[flat_token] : -1;
      const int see = pos >= 0 ? pos : INT_MAX;      // absent rows need no mask: nothing of theirs is written
      const int low = __reduce_min_sync(0xffffffffu, see);
      float m = kNegInf, l = 0.f;
      const int stride = dual ? 1 : 2;
      int begun = 0;
      for (int tile = s.begin + (dual ? 0 : w); tile < s.end; tile += stride, ++begun) {
        const uint32_t step = step0 + (dual ? 2 * begun + w : tile - s.begin);
        const uint32_t buf = step % kBufs;
        const uint32_t s_addr = lane_addr + buf * 128;
        if (!__all_sync(0xffffffffu, wait_tight(&sm.s_full[buf], step / kBufs & 1, abort, err, kSiteSFull))) {
          ok = false;
          break;
        }
        tc_fence_after();
        float x[kTile];
#pragma unroll
        for (int c = 0; c < kTile; c += 32) {
          uint32_t r[32];
          tmem_ld32(s_addr + c, r);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[c + i] = __uint_as_float(r[i]);
        }
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < kTile; ++c) asm volatile("" : "+f"(x[c]));   // no use before the wait
        const int key0 = tile * kTile;
        if (key0 + kTile - 1 > low || key0 + kTile > s.limit) {
          const int last = min(see, s.limit - 1) - key0;
#pragma unroll
          for (int c = 0; c < kTile; ++c)
            if (c > last) x[c] = kNegInf;
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < kTile - 4; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3(top[i], x[c + i], x[c + 4 + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], x[kTile - 4 + i]);
        const float peak = reference_point(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), p.scale_log2, kBelow);
        float alpha = 1.f;
        // A warp that has to rescale for one row takes the maxima of all its rows over.
        const bool outgrown = __any_sync(0xffffffffu, peak > m + kRescale<T> || (m == kNegInf && peak > m));
        if (outgrown && peak > m) {
          alpha = ex2(m - peak);     // 0 at the first key
          m = peak;
        }
        if (begun > 0 && outgrown) {
          if (!product_done()) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t r[16];
            tmem_ld16(o_addr + c, r);
            tc_wait_ld();
            hold(r);
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st16(o_addr + c, r);
          }
        }
        const float ref = finite_or_zero(m);
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), shift2 = make_float2(-ref, -ref);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < kTile; c += 32) {
          uint32_t packed[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 e = fma2(make_float2(x[c + 2 * i], x[c + 2 * i + 1]), scale2, shift2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[i & 1] = add2(sum[i & 1], e);
            packed[i] = pack2<T>(e.x, e.y);   // weights rounded for the second product, their sum is not
          }
          tmem_st16(s_addr + c / 2, packed);
          if (kHalves && c == kTile / 2 - 32) {
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&sm.p_half[buf]);
          }
        }
        sum[0] = add2(sum[0], sum[1]);
        l = l * alpha + (sum[0].x + sum[0].y);
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&sm.p_full[buf]);
        ++done;
      }
      if (!ok) break;
      step0 += (dual ? 2 : 1) * (s.end - s.begin);
      if (begun > 0) {
        if (!product_done()) break;
        tc_fence_after();
      }
      if (pos < 0) {   // a padding row: zero, no weight
        m = kNegInf;
        l = 0.f;
      }
      float other_m = kNegInf, other_l = 0.f;
      if (!dual) {
        // Warpgroup 1 leaves its statistics; warpgroup 0 reads both accumulators and writes.
        if (w == 1) {
          sm.ml[row][0] = begun > 0 ? m : kNegInf;
          sm.ml[row][1] = begun > 0 ? l : 0.f;
        }
        if (!join()) break;
        if (w == 0) {
          other_m = sm.ml[row][0];
          other_l = sm.ml[row][1];
        }
      }
      if (dual || w == 0) {
        const bool two = !dual && s.end - s.begin > 1;
        const float best = fmaxf(m, other_m), ref = finite_or_zero(best);
        float f0 = ex2(m - ref), f1 = ex2(other_m - ref);
        const float total = f0 * l + f1 * other_l;
        const bool write = present, whole = s.slot < 0;
        if (whole) {
          const float inv = total == 0.f ? 0.f : 1.f / total;
          f0 *= inv;
          f1 *= inv;
        }
        const int qhead = s.head * p.group + row % p.group;
        T* dst = static_cast<T*>(p.out) + ((present ? flat_token : 0) * p.heads + qhead) * D;
        const int64_t part = static_cast<int64_t>(s.slot) * p.row_tile + first * p.group + row;
        if (!whole && write) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(best, total);
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          uint32_t r[32];
          if (s.begin < s.end) {
            tmem_ld32(o_addr + c, r);
            tc_wait_ld();
            hold(r);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = pos >= 0 ? __uint_as_float(r[i]) * f0 : 0.f;
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (two) {
            tmem_ld32(o_addr + D + c, r);
            tc_wait_ld();
            hold(r);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] += pos >= 0 ? __uint_as_float(r[i]) * f1 : 0.f;
          }
          if (write && whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(dst + c + i) =
                  make_uint4(pack2<T>(o[i], o[i + 1]), pack2<T>(o[i + 2], o[i + 3]), pack2<T>(o[i + 4], o[i + 5]),
                             pack2<T>(o[i + 6], o[i + 7]));
          } else if (write) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(p.part_o + part * D + c + i) =
                  make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      tc_fence_before();
      if (!dual && !join()) break;   // accumulators and statistics have been read
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int D>
void launch(Args& args, int sms, cudaStream_t stream) {
  const Split split(args, sms, 0, kItemCost);
  constexpr bool kHalf = std::is_same_v<T, __half>;
  const CUtensorMap tq = make_query_map(args, kHalf, kM / args.group);
  const CUtensorMap tk = make_pool_map(args, args.k, kHalf, kTile);
  const CUtensorMap tv = make_pool_map(args, args.v, kHalf, kTile);
  const size_t smem = sizeof(ChunkSmem<D>) + 1024;
  auto kernel = paged_chunk_kernel<T, D>;
  allow_smem(reinterpret_cast<const void*>(kernel), smem);
  kernel<<<split.ctas, kThreads, smem, stream>>>(tq, tk, tv, args, device_error_slot(at::cuda::current_device()));
  EB_CUDA_CHECK(cudaGetLastError());
  count_launch(1);
  split.combine<T>(args, stream);
}

}  // namespace

template <typename T>
void paged_chunk_launch(Args& args, int sms, cudaStream_t stream) {
  set_rows(args, kM, kTile);
  // Two MMAs' rows an item when there are more than one MMA's.
  const int half_tokens = kM / args.group;
  args.tile_tokens = std::min(args.tokens, 2 * half_tokens);
  args.row_tile = args.tile_tokens * args.group;
  args.row_tiles = cdiv(args.tokens, args.tile_tokens);
  if (args.dim == 64) return launch<T, 64>(args, sms, stream);
  return launch<T, 128>(args, sms, stream);
}

template void paged_chunk_launch<__half>(Args&, int, cudaStream_t);
template void paged_chunk_launch<__nv_bfloat16>(Args&, int, cudaStream_t);

}  // namespace eb
