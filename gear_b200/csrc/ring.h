// Places in rings of mbarriers, and the phases to wait for.  No CUDA in here: the rules are tested on the host.
#pragma once

#ifdef __CUDACC__
#define GEARB_RING_FN __host__ __device__ __forceinline__
#else
#define GEARB_RING_FN inline
#endif

namespace gearb {
namespace rec {

// A place in a ring of barriers, and the parity of its use.
template <unsigned kSize>
struct Turn {
  unsigned i = 0, parity = 0;
  GEARB_RING_FN void next() {
    if (++i == kSize) {
      i = 0;
      parity ^= 1u;
    }
  }
};

// Whether `t` is the place of turn m, where it is known to be less than 2 * kSize turns away.
template <unsigned kSize>
GEARB_RING_FN bool is_turn(const Turn<kSize> &t, unsigned m) {
  return t.i == m % kSize && t.parity == (m / kSize & 1u);
}

// Waits for the phase of every turn, in order.  A wait knows the parity of a phase only: while the phase of kSize turns
// ago runs, that of 2 * kSize turns ago looks like this turn's, ended.  So no turn may be left out, not even one whose
// data is not needed.  (Waiting for the phase before first would not do: when this turn's has ended already, that one
// looks like the next, which cannot end yet.)
template <unsigned kSize>
struct Follower {
  Turn<kSize> turn;
  // wait(place, parity): as mbarrier.try_wait.parity in a loop; false when its limit ran out
  template <typename Wait>
  GEARB_RING_FN bool pass(Wait &&wait) {
    const bool ended = wait(turn.i, turn.parity);
    turn.next();
    return ended;
  }
};

}  // namespace rec
}  // namespace gearb
