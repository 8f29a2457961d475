// Phases of the barriers that the chunk kernel's products complete, apart from the
// kernel so that a host program can go through every state they can be in.
//
// A parity wait tells a finished phase n from a pending one only while phase n - 1 is
// known to be complete: two phases back reads like complete, and waiting for phase
// n - 1 when n is complete as well never ends. Seeing the scores of step i, a softmax
// warpgroup knows that the products up to step i - (score buffers) are complete. With
// three buffers that leaves its last but one product open, so at an item's end two of
// its products may be pending. Two barriers a warpgroup, taken in turn, have one
// pending phase each, whatever finishes when.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define EB_PHASE_FN __host__ __device__ __forceinline__
#else
#define EB_PHASE_FN inline
#endif

namespace eb {
namespace paged {

constexpr uint32_t kProductBarriers = 2;   // of a warpgroup

struct Phase {
  uint32_t barrier, parity;
};

// Barrier and parity that say whether a warpgroup's product n (0 is the launch's first) is complete.
EB_PHASE_FN Phase product_phase(uint32_t n) { return {n % kProductBarriers, n / kProductBarriers & 1}; }

}  // namespace paged
}  // namespace eb
