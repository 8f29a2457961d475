// Phases of the chunk kernel's barriers, apart from the kernel so that a host program
// can go through every state they can be in.
//
// Products.
// A parity wait tells a finished phase n from a pending one only while phase n - 1 is
// known to be complete: two phases back reads like complete, and waiting for phase
// n - 1 when n is complete as well never ends. Seeing the scores of step i, a softmax
// warpgroup knows that the products up to step i - (score buffers) are complete. With
// three buffers that leaves its last but one product open, so at an item's end two of
// its products may be pending. Two barriers a warpgroup, taken in turn, have one
// pending phase each, whatever finishes when.
//
// Copies. Each operand counts its own copies, so that a CTA that gives up between the
// keys and the values of a tile waits for all that it has under way before it exits.
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

// Copies of one operand into a ring of `stages` slots, copy n into slot n % stages.
struct CopyRing {
  uint32_t issued = 0;

  // Slot of the next copy, and the parity of its barriers' phase that the copy completes.
  EB_PHASE_FN Phase next(uint32_t stages) const { return {issued % stages, issued / stages & 1}; }
  // The next copy's slot has held another one: wait until that has been read (parity next().parity ^ 1).
  EB_PHASE_FN bool reuses(uint32_t stages) const { return issued >= stages; }

  // Calls wait(slot, parity) for every copy that may still be under way.
  template <typename F>
  EB_PHASE_FN void drain(uint32_t stages, F wait) const {
    for (uint32_t n = issued > stages ? issued - stages : 0; n < issued; ++n) wait(n % stages, n / stages & 1);
  }
};

}  // namespace paged
}  // namespace eb
