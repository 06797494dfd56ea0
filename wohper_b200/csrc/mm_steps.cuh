// mm_steps.cuh -- by which steps the warps of the FP8 product (fp8_gemm.cu) wait for one
// another: the barrier and phase before a stage of its ring is filled, and what an
// epilogue's warps do together.  Plain C++: CPU tests compile it too, and run through
// every order in which the warps can come and through waits that run out.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define WH_STEP __device__ __forceinline__
#else
#define WH_STEP inline
#endif

namespace wh {

// Tile f's products, done, arrive on barrier bar(f) and end its phase of parity(f);
// tile f + kStages, which takes the same stage, is filled after that.
// A wait by parity tells a phase from its two neighbours only.
//  - kBars == kStages, for a warp that fills every tile: the phase after the awaited one
//    is that of the tile it is about to fill.
//  - kBars == 2 * kStages, for warps that take a stage's tiles in turn: one may come to its
//    wait when the other's tile has been filled and multiplied as well.  On kStages barriers
//    that is a phase too late, and the wait then lasts until its limit; here the phase
//    after the awaited one is tile f + 2 * kStages's, which follows tile f + kStages in its
//    stage, the one the warp is about to fill.
template <int kStages, int kBars>
struct MmFree {
  static_assert(kBars == kStages || kBars == 2 * kStages, "one phase ahead at most");
  static WH_STEP int bar(int f) { return f % kBars; }
  static WH_STEP uint32_t parity(int f) { return uint32_t(f / kBars) & 1u; }
};

// One tile of an epilogue warp: `sum` takes each of its sums from the tensor core (false:
// the wait ran out), `store` writes the tile together with the other warps of its column half.
// Those wait for one another without a limit, so the warps `agree` first: all of them store
// the tile or, where one has given up, none.
template <class Sum, class Agree, class Store>
WH_STEP bool mm_tile(int ktiles, int fold, Sum sum, Agree agree, Store store) {
  bool ok = true;
  for (int c0 = 0; ok && c0 < ktiles; c0 += fold) ok = sum(c0 == 0);
  ok = agree(ok);
  if (ok) store();
  return ok;
}

}  // namespace wh
