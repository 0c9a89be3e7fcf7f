// The ring of key and value chunks of the prompts' kernel, and the order in which its producer
// fills it.  Plain C++ as well, so that a host test can run the order as it stands.
//
// A CTA's g-th key tile has its keys in chunks 5 g .. 5 g + 2 of the ring and its values behind the
// next tile's keys.  So what a chunk takes the place of is: K_g, of K_g-2's last chunk and V_g-3;
// V_g, of K_g's first two.  Each of the ring's barriers ("keys in", "values in", ...) exists twice, for
// even and odd tiles, and a copy into one of them may be announced only when the copy before it on the same
// barrier has arrived and whoever waits for that one has seen it.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define NTB200_RING __host__ __device__ __forceinline__
#else
#define NTB200_RING inline
#endif

namespace ntb200 {

constexpr uint32_t kRingKeys = 3, kRingValues = 2, kRingChunks = 8;

NTB200_RING constexpr uint32_t k_chunk(uint32_t g) { return g * (kRingKeys + kRingValues); }
NTB200_RING constexpr uint32_t v_chunk(uint32_t g) { return k_chunk(g + 1) + kRingKeys; }

// Ops, each of them for key tile g:
//   bool keys_half_used(g)  waits until the products with the keys' first two chunks are complete
//   bool keys_used(g)       ... with all of them
//   bool values_used(g)     ... with the values
//   void load_keys(g), void load_values(g)
// A wait that gave up is false and ends the filling.
struct RingFill {
  uint32_t nk = 0, nv = 0;  // key tiles, value tiles loaded

  // The next tile's keys.  V_nk-3's copy has arrived and been seen once its products are complete; so
  // has K_nk-2's, the one before on this barrier.
  template <typename Ops>
  NTB200_RING bool keys(Ops& ops) {
    if (nk >= 3 && !ops.values_used(nk - 3)) return false;
    if (nk >= 2 && !ops.keys_used(nk - 2)) return false;
    ops.load_keys(nk++);
    return true;
  }

  // Values that stay a tile behind the keys.  keys() has waited for V_nv-2, the copy before on this barrier.
  template <typename Ops>
  NTB200_RING bool values_behind(Ops& ops) {
    if (nv + 1 >= nk) return true;
    if (!ops.keys_half_used(nv)) return false;
    ops.load_values(nv++);
    return true;
  }

  // The last tile's values.  No keys() came in between, and where only one tile of rows visits the last key
  // tile its keys may be used up while V_nv-2 is still on its way.
  template <typename Ops>
  NTB200_RING bool last_values(Ops& ops) {
    if (nv >= nk) return true;
    if (nv >= 2 && !ops.values_used(nv - 2)) return false;
    if (!ops.keys_half_used(nv)) return false;
    ops.load_values(nv++);
    return true;
  }
};

}  // namespace ntb200
