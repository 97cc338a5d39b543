// A follower of a ring of modelled mbarriers, in every state that a tile of the streaming recurrences may find the ring in.
// Exit code 0: every wait of a follower that takes every turn ended behind the phase it was for and none was left
// waiting, and the model sees that leaving turns out goes wrong.
#include <cstdio>

#include "ring.h"

using gearb::rec::Follower;

constexpr unsigned kRing = 3;

// Phases of the ring's barriers end turn after turn.  A wait that does not end lets the next turn end, up to the last
// one that can while the waiter waits.
struct Model {
  unsigned ended, last;  // turns whose phase has ended; how many can
  unsigned at(unsigned place) const { return ended > place ? (ended - place - 1) / kRing + 1 : 0; }  // phases of a barrier
  bool wait(unsigned place, unsigned parity) {
    while ((at(place) & 1u) == parity) {  // the running phase has it: the one before does not
      if (ended == last) return false;
      ++ended;
    }
    return true;
  }
};

// Waits at every `every`-th of 60 tiles; states in which a wait went wrong.
unsigned faults(unsigned stages, unsigned every, unsigned &checked) {
  unsigned bad = 0, sure = 0;  // turns known to have ended
  Follower<kRing> follower;
  for (unsigned m = 0; m < 60; ++m) {
    // Tile m has arrived, so tile m - stages has left.  Tiles before m have been let go and two more are looked at in front
    // of them, so the phases of at most m + 2 turns have ended.
    const unsigned left = m >= stages ? m - stages + 1 : 0;
    if (m % every != every - 1) {
      follower.turn.next();
      continue;
    }
    const Follower<kRing> before = follower;
    for (unsigned ended = left > sure ? left : sure; ended <= m + 2; ++ended) {
      Model model{ended, m + 2};
      follower = before;
      const bool ok = follower.pass([&](unsigned place, unsigned parity) { return model.wait(place, parity); });
      bad += !ok || model.ended <= m;
      ++checked;
    }
    sure = m + 1;
  }
  return bad;
}

// Two recorders take every other turn and leave the place of the first that they have not recorded.  Turns [from, to) are
// gone through as a launch that gives up does: which of them has its recorder left out?
template <unsigned kStages>
bool left_out_is_found(unsigned &checked) {
  constexpr unsigned kRecorders = 2;
  for (unsigned from = 0; from < 60; ++from)
    for (unsigned to = from; to <= from + kStages; ++to)
      for (unsigned r = 0; r < kRecorders; ++r)
        for (unsigned first = from + (from % kRecorders != r); first <= to + 1; first += kRecorders) {
          gearb::rec::Turn<kStages> place;
          for (unsigned k = 0; k < first; ++k) place.next();
          bool recorded = true;
          for (unsigned m = from; m < to; ++m) {
            if (m % kRecorders != r) continue;
            if (gearb::rec::is_turn(place, m)) recorded = false;
            if (recorded != (m < first)) return false;
            ++checked;
          }
        }
  return true;
}

int main() {
  unsigned checked = 0;
  if (!left_out_is_found<4>(checked) || !left_out_is_found<5>(checked) || !left_out_is_found<6>(checked)) {
    std::printf("a turn that was not recorded is taken for one that was, or the other way round\n");
    return 1;
  }
  for (unsigned stages = 4; stages <= 6; ++stages) {
    if (faults(stages, 1, checked) != 0) {
      std::printf("%u stages: a wait ended early, or never\n", stages);
      return 1;
    }
    if (faults(stages, 8, checked) == 0) {
      std::printf("%u stages: the model does not see turns left out\n", stages);
      return 1;
    }
  }
  std::printf("%u states ok\n", checked);
  return 0;
}
