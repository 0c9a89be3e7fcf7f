// Which phase of which barrier tells that the paged prefill's g-th product O += P_g V_g is complete.
// Plain C++ as well, so that a host test can check every wait for it.
//
// A wait by parity tells phase n from n - 1 only, so whoever waits for phase n has to know already that
// n - 1 is over.  The softmax waits for a product only where it rescales O and at an item's end, and knows
// no more than what its scores S_g tell: that product g - 2 is complete, which S_g's issuer has waited for.
// So products alternate between two barriers, on which g - 2 comes right before g.  (With one barrier for all
// of them an item's end was taken for reached while the product before its last was still to come, and O
// was read too early.)
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define NTB200_PHASES __host__ __device__ __forceinline__
#else
#define NTB200_PHASES inline
#endif

namespace ntb200 {

struct ProductPhase {
  uint32_t barrier, parity;
};

NTB200_PHASES constexpr ProductPhase product_phase(uint32_t g) { return {g & 1, (g >> 1) & 1}; }

}  // namespace ntb200
