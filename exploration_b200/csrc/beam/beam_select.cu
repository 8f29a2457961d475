// Beam search's selection: the best `beams` continuations of a group of beams.
//
// Beam w at cumulative score c_w offers token t at c_w + (x_wt - lse_w) with
// lse_w = log sum_t exp(x_wt); an ended beam offers only (eos, c_w). With the
// beam's largest logit m the difference is taken as (x_wt - m) - log sum_t
// exp(x_wt - m), so that neither large logits nor a mask of the type's lowest
// value (whose product with log2(e) is infinite) cost it any bits. Inside a
// beam candidates are ordered by logit, then by token; across beams by score,
// then by beam: rounding of the sum never reorders a beam's tokens, so each
// beam's best `beams` logits are all that the final choice needs. A beam whose
// lse is not finite (nothing left unmasked, or a NaN) offers tokens 0, 1, ... at -inf.
//
// Bound by one read of the logits (and by latency below a few MB). A warp holds
// 1,024 logits in registers and takes its maximum, sum and best K from there
// (redux.sync on order-preserving integers). Up to 1,024 tokens one CTA a group
// with a warp a beam does all in one launch. Longer rows are cut into chunks of
// 8,192, one CTA each, whose sums and best K a second, overlapped launch joins:
// sums of chunks in fp64, so they do not depend on the cut beyond a rounding.
// Measured: 8 x 8 beams of 100,003 bf16 logits (12.8 MB): 15.5 us for the chunks
// (700 instructions a warp; 39 us when every round searched all logits), 26 us in all;
// 4 x 4 beams of 256 tokens: 4.3 us of kernel.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <climits>

#include "../common/checks.h"
#include "../common/util.cuh"

namespace eb {
namespace {

constexpr int kPerLane = 32;
constexpr int kWarpTokens = 32 * kPerLane;
constexpr int kChunkWarps = 8;
constexpr int kChunk = kChunkWarps * kWarpTokens;
constexpr int kMaxBeams = 32;
constexpr int kList = 64;           // candidates of a warp
constexpr int kJoinWarps = 8;
constexpr int kHeld = 8;            // candidates a lane of the joining warp holds
constexpr float kLog2e = 1.4426950408889634f;

struct SelectArgs {
  const void* logits;        // [rows, vocab], dense
  const float* scores;       // [rows]
  const bool* finished;
  float* scores_out;
  int64_t* parents;
  int64_t* tokens;
  bool* finished_out;
  float* part_ms;            // [rows, chunks, 2]
  float* part_x;             // [rows, chunks, beams]
  int* part_t;
  int beams, vocab, chunks, keep, eos;   // keep = min(beams, vocab)
};

// Order-preserving map of floats to unsigned integers.
EB_DEVICE uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
EB_DEVICE float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// Calls take(round, value, token) in every lane for the best `count` of the warp's
// 64-bit keys (ordered value, inverted token; 0: none).
template <int N, typename F>
EB_DEVICE void pick_from(int count, uint64_t (&keys)[N], F take) {
  for (int round = 0; round < count; ++round) {
    uint64_t high = keys[0];
#pragma unroll
    for (int i = 1; i < N; ++i) high = keys[i] > high ? keys[i] : high;
    const uint32_t value = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(high >> 32));
    const uint32_t low = static_cast<uint32_t>(high >> 32) == value ? static_cast<uint32_t>(high) : 0u;
    const uint32_t first = __reduce_max_sync(0xffffffffu, low);
    take(round, unordered(value), value == 0 ? INT_MAX : static_cast<int>(0xffffffffu - first));
    const uint64_t gone = static_cast<uint64_t>(value) << 32 | first;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (keys[i] == gone) keys[i] = 0;
  }
}

template <typename F>
EB_DEVICE void pick(int count, uint64_t a, uint64_t b, F take) {
  uint64_t keys[2] = {a, b};
  pick_from(count, keys, take);
}

// A lane's logits: kPerLane / VE vectors, vector j at index (j * 32 + lane) * VE of
// the warp's span. Absent ones are -inf. `begin` may lie before the row (alignment).
template <typename T>
struct LaneLogits {
  static constexpr int VE = 16 / sizeof(T);
  float x[kPerLane];
  int64_t begin;   // token index of the warp's span

  EB_DEVICE int token(int i, int lane) const {
    return static_cast<int>(begin) + ((i / VE) * 32 + lane) * VE + i % VE;
  }

  EB_DEVICE void load(const T* row, int64_t from, int vocab, int lane) {
    begin = from;
#pragma unroll
    for (int j = 0; j < kPerLane / VE; ++j) {
      const int64_t t = from + (j * 32 + lane) * VE;
      if (t >= 0 && t + VE <= vocab) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + t);
        const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < VE; ++i) x[j * VE + i] = load_f<T>(h + i);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) 
          x[j * VE + i] = t + i >= 0 && t + i < vocab ? load_f<T>(row + t + i) : kNegInf;
      }
    }
  }

  // Maximum and sum of exp(x - max) over the warp; `peak`: of this lane alone.
  EB_DEVICE void sum(float& m, float& s, float& peak) const {
    peak = kNegInf;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) peak = fmaxf(peak, x[i]);
    m = warp_max(peak);
    const float ref = finite_or_zero(m);
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) part[i & 1] += ex2((x[i] - ref) * kLog2e);
    s = warp_sum(part[0] + part[1]);
  }

  // Bits of this lane's logits that exist.
  EB_DEVICE uint32_t present(int vocab, int lane) const {
    if (begin >= 0 && begin + kWarpTokens <= vocab) return 0xffffffffu;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int t = token(i, lane);
      bits |= static_cast<uint32_t>(t >= 0 && t < vocab) << i;
    }
    return bits;
  }

  // Calls take(round, value, token) in every lane for the best `count` logits in order
  // (token INT_MAX: no more). The count-th largest of the lanes' maxima bounds the
  // count-th logit from below, so only the few logits that reach it are looked at
  // further: they are read again and gathered into `list` (shared memory of this
  // warp). Should few lanes hold too many of them, every round goes through all logits.
  template <typename F>
  EB_DEVICE void best(int count, int vocab, int lane, const T* row, float peak, uint64_t* list, F take) const {
    const uint32_t valid = present(vocab, lane);
    const uint32_t top = valid ? ordered(peak + 0.f) : 0u;   // -0 ties with 0; 0: below every float's key
    uint32_t bound = top, left = top;
    for (int round = 0; round < count; ++round) {
      bound = __reduce_max_sync(0xffffffffu, left);
      // One lane leaves the race; equal maxima count one by one.
      if (lane == __ffs(__ballot_sync(0xffffffffu, left == bound)) - 1) left = 0;
    }
    bound = max(bound, ordered(kNegInf));
    uint32_t above = 0, equal = 0;
    if (top >= bound) {
      const float limit = unordered(bound);
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        above |= static_cast<uint32_t>(x[i] > limit) << i;
        equal |= static_cast<uint32_t>(x[i] == limit) << i;
      }
      above &= valid;
      equal &= valid;
    }
    // Place of this lane's n entries among the warp's, and their total.
    auto place = [&](int n, int& all) {
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      all = __shfl_sync(0xffffffffu, upto, 31);
      return upto - n;
    };
    // Value first, then the lower token: one 64-bit key.
    auto entry = [&](uint32_t k, int t) {
      return static_cast<uint64_t>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(t));
    };
    int total;
    int at = place(__popc(above), total);
    if (total + count <= kList) {
      for (; above; above &= above - 1) {
        const int t = token(__ffs(above) - 1, lane);
        list[at++] = entry(ordered(load_f<T>(row + t) + 0.f), t);
      }
      // Of the logits equal to the bound (all of a masked stretch, perhaps) the first `count` tokens.
      const int limit = total + count;
#pragma unroll 1
      for (int j = 0; j < kPerLane / VE && total < limit; ++j) {
        uint32_t mine = equal >> (j * VE) & ((1u << VE) - 1);
        if (!__any_sync(0xffffffffu, mine != 0)) continue;
        int all;
        int slot = total + place(__popc(mine), all);
        for (; mine && slot < limit; mine &= mine - 1) list[slot++] = entry(bound, token(j * VE + __ffs(mine) - 1, lane));
        total += all;
      }
      total = min(total, limit);
      __syncwarp();
      pick(count, lane < total ? list[lane] : 0, lane + 32 < total ? list[lane + 32] : 0, take);
      __syncwarp();
      return;
    }
    uint32_t last_key = 0xffffffffu;
    int last_token = -1;
    for (int round = 0; round < count; ++round) {
      uint32_t key = 0;
      int t_best = INT_MAX;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int t = token(i, lane);
        const uint32_t k = ordered(x[i] + 0.f);
        const bool after = k < last_key || (k == last_key && t > last_token);   // not taken yet
        if ((valid >> i & 1) && after && (t_best == INT_MAX || k > key)) {
          key = k;
          t_best = t;
        }
      }
      const uint32_t value = __reduce_max_sync(0xffffffffu, t_best == INT_MAX ? 0u : key);
      const int first = __reduce_min_sync(0xffffffffu, t_best != INT_MAX && key == value ? t_best : INT_MAX);
      take(round, unordered(value), first);
      last_key = value;
      last_token = first;
    }
  }
};

// Token index of the first 16-byte boundary at or before `row`'s chunk start.
template <typename T>
EB_DEVICE int64_t aligned_start(const T* row) {
  constexpr int VE = 16 / sizeof(T);
  const int ahead = static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VE);
  return -ahead;
}

// One warp: the best `beams` of the beams' sorted candidate lists total[w][i], token[w][i] (shared memory).
EB_DEVICE void choose(const SelectArgs& p, int group, int lane, const float (*total)[kMaxBeams],
                      const int (*token)[kMaxBeams]) {
  int at = 0;
  const bool ended = lane < p.beams && p.finished[group * p.beams + lane];
  for (int round = 0; round < p.beams; ++round) {
    const bool live = lane < p.beams && at < p.keep;
    const uint32_t key = live ? ordered(total[lane][at] + 0.f) : 0u;
    const uint32_t top = __reduce_max_sync(0xffffffffu, key);
    const int winner = __ffs(__ballot_sync(0xffffffffu, live && key == top)) - 1;
    if (lane == winner) {
      const int64_t out = static_cast<int64_t>(group) * p.beams + round;
      p.scores_out[out] = total[lane][at];
      p.parents[out] = lane;
      p.tokens[out] = token[lane][at];
      p.finished_out[out] = ended || token[lane][at] == p.eos;
      ++at;
    }
  }
}

// Candidate i of a beam with logit x, largest logit m and log_sum = log sum exp(x - m): its total score.
EB_DEVICE void offer(const SelectArgs& p, float base, bool ended, float m, float log_sum, int i, float x, int t,
                     float& total, int& token) {
  if (ended) {
    total = i == 0 ? base : kNegInf;
    token = p.eos;
  } else if (!isfinite(m) || !isfinite(log_sum)) {
    total = kNegInf;
    token = i;
  } else {
    const float sum = __fadd_rn(base, __fsub_rn(__fsub_rn(x, m), log_sum));
    total = sum == sum ? sum : kNegInf;
    token = t;
  }
}

// Up to kWarpTokens tokens: one CTA a group, one warp a beam.
template <typename T>
__global__ void __launch_bounds__(1024)
beam_select_small_kernel(SelectArgs p) {
  __shared__ float total[kMaxBeams][kMaxBeams];
  __shared__ int token[kMaxBeams][kMaxBeams];
  __shared__ uint64_t list[kMaxBeams][kList];
  const int group = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = group * p.beams + warp;
  {
    const T* logits = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.vocab;
    LaneLogits<T> x;
    x.load(logits, aligned_start(logits), p.vocab, lane);
    const float score = p.scores[row];
    const bool ended = p.finished[row];
    float m, s, peak;
    x.sum(m, s, peak);
    const float log_sum = logf(s);
    x.best(p.keep, p.vocab, lane, logits, peak, list[warp], [&](int i, float value, int t) {
      if (lane == 0) offer(p, score, ended, m, log_sum, i, value, t, total[warp][i], token[warp][i]);
    });
  }
  __syncthreads();
  if (warp == 0) choose(p, group, lane, total, token);
}

// Longer rows, first launch: sums and best K of one chunk.
template <typename T>
__global__ void __launch_bounds__(kChunkWarps * 32, 3)
beam_select_chunk_kernel(SelectArgs p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining CTAs may be set up
  __shared__ float sm_m[kChunkWarps], sm_s[kChunkWarps];
  __shared__ float sm_x[kChunkWarps][kMaxBeams];
  __shared__ int sm_t[kChunkWarps][kMaxBeams];
  __shared__ uint64_t list[kChunkWarps][kList];
  const int chunk = blockIdx.x, row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* logits = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.vocab;
  {
    LaneLogits<T> x;
    x.load(logits, aligned_start(logits) + static_cast<int64_t>(chunk) * kChunk + warp * kWarpTokens, p.vocab, lane);
    float m, s, peak;
    x.sum(m, s, peak);
    if (lane == 0) {
      sm_m[warp] = m;
      sm_s[warp] = s;
    }
    x.best(p.keep, p.vocab, lane, logits, peak, list[warp], [&](int i, float value, int t) {
      if (lane == 0) {
        sm_x[warp][i] = value;
        sm_t[warp][i] = t;
      }
    });
  }
  __syncthreads();
  if (warp != 0) return;
  const int64_t part = static_cast<int64_t>(row) * p.chunks + chunk;
  float m = lane < kChunkWarps ? sm_m[lane] : kNegInf;
  const float top = warp_max(m), ref = finite_or_zero(top);
  const float s = warp_sum(lane < kChunkWarps ? sm_s[lane] * ex2((m - ref) * kLog2e) : 0.f);
  if (lane == 0) {
    p.part_ms[part * 2] = top;
    p.part_ms[part * 2 + 1] = s;
  }
  int at = 0;
  for (int round = 0; round < p.keep; ++round) {
    const bool live = lane < kChunkWarps && at < p.keep && sm_t[lane][at] != INT_MAX;
    const uint32_t key = live ? ordered(sm_x[lane][at]) : 0u;
    const uint32_t best = __reduce_max_sync(0xffffffffu, key);
    // Lower warps hold lower tokens: the first of equal logits is the lowest token.
    const int winner = __ffs(__ballot_sync(0xffffffffu, live && key == best)) - 1;
    if (winner < 0) {
      if (lane == 0) {
        p.part_x[part * p.keep + round] = kNegInf;
        p.part_t[part * p.keep + round] = INT_MAX;
      }
    } else if (lane == winner) {
      p.part_x[part * p.keep + round] = sm_x[lane][at];
      p.part_t[part * p.keep + round] = sm_t[lane][at];
      ++at;
    }
  }
}

// One warp: a beam's sums and best logits from its chunks'.
EB_DEVICE void join_beam(const SelectArgs& p, int row, int lane, float* total, int* token) {
  const int64_t base = static_cast<int64_t>(row) * p.chunks;
  // Everything that the beam needs is read at once.
  const float score = p.scores[row];
  const bool ended = p.finished[row];
  const int entries = p.chunks * p.keep;
  uint64_t keys[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int e = i * 32 + lane;
    keys[i] = 0;
    if (e < entries) {
      const int t = p.part_t[base * p.keep + e];
      const float v = p.part_x[base * p.keep + e];
      if (t != INT_MAX)
        keys[i] = static_cast<uint64_t>(ordered(v + 0.f)) << 32 | (0xffffffffu - static_cast<uint32_t>(t));
    }
  }
  float m = kNegInf;
  for (int c = lane; c < p.chunks; c += 32) m = fmaxf(m, p.part_ms[(base + c) * 2]);
  m = warp_max(m);
  const float ref = finite_or_zero(m);
  // The chunks' sums are added in fp64: the result depends on the cut by no more than its own rounding.
  double sum = 0.0;
  for (int c = lane; c < p.chunks; c += 32) {
    const float2 ms = *reinterpret_cast<const float2*>(p.part_ms + (base + c) * 2);
    sum += static_cast<double>(ms.y * ex2((ms.x - ref) * kLog2e));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float log_sum = logf(static_cast<float>(sum));
  if (entries <= 32 * kHeld) {
    pick_from(p.keep, keys, [&](int i, float value, int t) {
      if (lane == 0) offer(p, score, ended, m, log_sum, i, value, t, total[i], token[i]);
    });
    return;
  }
  // Longer: K rounds over the chunks' sorted lists, chunk c with lane c % 32.
  uint32_t key = 0;
  int mine = INT_MAX;
  // A lane with several chunks rescans their lists for its best entry after (last value, last token).
  uint32_t last_key = 0xffffffffu;
  int last_t = -1;
  auto rescan = [&]() {
    key = 0;
    mine = INT_MAX;
    for (int c = lane; c < p.chunks; c += 32) {
      for (int i = 0; i < p.keep; ++i) {
        const int t = p.part_t[(base + c) * p.keep + i];
        if (t == INT_MAX) break;
        const uint32_t k = ordered(p.part_x[(base + c) * p.keep + i]);
        if (k > last_key || (k == last_key && t <= last_t)) continue;   // taken before
        if (mine == INT_MAX || k > key || (k == key && t < mine)) {
          key = k;
          mine = t;
        }
        break;
      }
    }
  };
  rescan();
  for (int round = 0; round < p.keep; ++round) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, mine == INT_MAX ? 0u : key);
    const int cand = mine != INT_MAX && key == top ? mine : INT_MAX;
    const int first = __reduce_min_sync(0xffffffffu, cand);
    if (lane == 0) offer(p, score, ended, m, log_sum, round, unordered(top), first, total[round], token[round]);
    if (cand == first && first != INT_MAX) {
      last_key = key;
      last_t = mine;
      rescan();
    }
  }
}

// Second launch: one CTA a group; warps take the beams in turn and join their chunks, then the choice.
__global__ void __launch_bounds__(kJoinWarps * 32)
beam_select_join_kernel(SelectArgs p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float total[kMaxBeams][kMaxBeams];
  __shared__ int token[kMaxBeams][kMaxBeams];
  const int group = blockIdx.x, lane = threadIdx.x & 31;
  for (int beam = threadIdx.x >> 5; beam < p.beams; beam += blockDim.x >> 5)
    join_beam(p, group * p.beams + beam, lane, total[beam], token[beam]);
  __syncthreads();
  if (threadIdx.x < 32) choose(p, group, lane, total, token);
}

template <typename T>
void launch(SelectArgs& args, int groups, const at::TensorOptions& f32, cudaStream_t stream) {
  if (args.vocab + 16 / static_cast<int>(sizeof(T)) - 1 <= kWarpTokens) {
    beam_select_small_kernel<T><<<groups, 32 * args.beams, 0, stream>>>(args);
    EB_CUDA_CHECK(cudaGetLastError());
    count_launch(1);
    return;
  }
  const int64_t rows = static_cast<int64_t>(groups) * args.beams;
  // One chunk more than the vocabulary needs when the row starts inside a vector.
  args.chunks = cdiv(args.vocab + 16 / static_cast<int>(sizeof(T)) - 1, kChunk);
  at::Tensor space = at::empty({rows * args.chunks * (2 + 2 * args.keep)}, f32);
  args.part_ms = space.data_ptr<float>();
  args.part_x = args.part_ms + rows * args.chunks * 2;
  args.part_t = reinterpret_cast<int*>(args.part_x + rows * args.chunks * args.keep);
  beam_select_chunk_kernel<T><<<dim3(args.chunks, rows), kChunkWarps * 32, 0, stream>>>(args);
  EB_CUDA_CHECK(cudaGetLastError());
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(groups);
  config.blockDim = dim3(32 * std::min(args.beams, kJoinWarps));
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  EB_CUDA_CHECK(cudaLaunchKernelEx(&config, beam_select_join_kernel, args));
  count_launch(2);
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> beam_select(const at::Tensor& logits_in,
                                                                       const at::Tensor& scores_in,
                                                                       const at::Tensor& finished_in, int64_t eos) {
  // The Python module makes the same checks for CPU tensors, with the same messages.
  TORCH_CHECK_VALUE(logits_in.dim() == 3 && scores_in.dim() == 2 && scores_in.size(0) == logits_in.size(0) &&
                        scores_in.size(1) == logits_in.size(1) && finished_in.sizes() == scores_in.sizes(),
                    "expected logits [groups, beams, vocab] and scores, finished [groups, beams]");
  TORCH_CHECK_VALUE(scores_in.scalar_type() == at::kFloat && finished_in.scalar_type() == at::kBool,
                    "scores must be fp32 and finished bool");
  TORCH_CHECK_VALUE(same_device(logits_in, scores_in, finished_in), "all tensors must be on one device");
  const int64_t groups = logits_in.size(0), beams = logits_in.size(1), vocab = logits_in.size(2);
  static_assert(kMaxBeams == 32);
  TORCH_CHECK_VALUE(beams >= 1 && beams <= kMaxBeams && vocab >= 1, "between 1 and 32 beams and at least one token");
  TORCH_CHECK_VALUE(!wants_grad(logits_in) && !wants_grad(scores_in),
                    "beam_select is for inference: it has no gradient");
  TORCH_CHECK_VALUE(eos >= -1 && eos < vocab, "eos must be a token or -1");
  TORCH_CHECK_VALUE(native_dtype(logits_in), "the native selection takes fp32, fp16 or bf16 logits");
  TORCH_CHECK(groups * beams < 65536 && vocab < (1LL << 30), "beam_select: too many rows or tokens");
  c10::cuda::CUDAGuard guard(logits_in.device());
  const at::Tensor logits = logits_in.contiguous(), scores = scores_in.contiguous(), finished = finished_in.contiguous();
  at::Tensor scores_out = at::empty_like(scores);
  at::Tensor both = at::empty({2, groups, beams}, scores.options().dtype(at::kLong));
  at::Tensor parents = both.select(0, 0), tokens = both.select(0, 1);
  at::Tensor finished_out = at::empty_like(finished);
  if (groups * beams > 0) {
    SelectArgs args{};
    args.logits = logits.data_ptr();
    args.scores = scores.data_ptr<float>();
    args.finished = finished.data_ptr<bool>();
    args.scores_out = scores_out.data_ptr<float>();
    args.parents = parents.data_ptr<int64_t>();
    args.tokens = tokens.data_ptr<int64_t>();
    args.finished_out = finished_out.data_ptr<bool>();
    args.beams = beams;
    args.vocab = vocab;
    args.keep = std::min(beams, vocab);
    args.eos = eos;
    auto stream = at::cuda::getCurrentCUDAStream();
    switch (logits.scalar_type()) {
      case at::kFloat: launch<float>(args, groups, scores.options(), stream); break;
      case at::kHalf: launch<__half>(args, groups, scores.options(), stream); break;
      case at::kBFloat16: launch<__nv_bfloat16>(args, groups, scores.options(), stream); break;
      default: TORCH_CHECK(false, "beam_select: fp32, fp16 or bf16 logits");
    }
  }
  return {scores_out, parents, tokens, finished_out};
}

}  // namespace eb
