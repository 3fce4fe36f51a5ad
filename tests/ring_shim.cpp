// immerdink_b200/csrc/common/ring.hpp against a model of a barrier on the host.
#include <vector>

#include "common/ring.hpp"

namespace {
// A barrier whose phases complete one after another, `done` so far: a question for a parity is answered yes unless the phase
// of that parity is the one that has still to complete.
struct Barrier {
  uint32_t armed = 0, done = 0;
  bool completed(uint32_t parity) const { return (done & 1u) != parity; }
};
}  // namespace

extern "C" {
// `issued` loads into a ring of `slots`; the last `open` of them (at most one a slot) land only at poll number `at` of the
// wait (never: 0). 0: as it should be; else what went wrong.
int ring_case(int slots, uint32_t issued, uint32_t open, uint32_t at) {
  std::vector<Barrier> bar(slots);
  for (uint32_t i = 0; i < issued; ++i) ++bar[i % slots].armed;
  for (uint32_t i = 0; i + open < issued; ++i) ++bar[i % slots].done;
  for (int s = 0; s < slots; ++s) {
    const int parity = imd::last_parity(issued, slots, s);
    if ((parity < 0) != (bar[s].armed == 0)) return 1;
    if (parity >= 0 && static_cast<uint32_t>(parity) != ((bar[s].armed - 1) & 1u)) return 2;
  }
  uint32_t polls = 0;
  const bool all = imd::await_ring(issued, slots, 64, [&](int s, uint32_t parity) {
    if (++polls == at)
      for (auto& b : bar) b.done = b.armed;
    return bar[s].completed(parity);
  });
  bool landed = true;
  for (const auto& b : bar) landed = landed && b.done == b.armed;
  if (all != landed) return 3;              // gave the memory back early, or waited for nothing
  if (at == 0 && open > 0 && all) return 4;
  if (open == 0 && polls > static_cast<uint32_t>(slots)) return 5;
  return polls <= 64u * slots ? 0 : 6;      // bounded
}

// The same without the number of loads: `open` of the slots (the first ones) wait for a copy.
int slots_case(int slots, uint32_t rounds, uint32_t open, uint32_t at) {
  std::vector<Barrier> bar(slots);
  for (int s = 0; s < slots; ++s) bar[s].done = rounds, bar[s].armed = rounds + (static_cast<uint32_t>(s) < open ? 1 : 0);
  uint32_t polls = 0;
  const bool all = imd::await_slots(slots, 64, [&](int s, uint32_t parity) {
    if (++polls == at)
      for (auto& b : bar) b.done = b.armed;
    return bar[s].completed(parity);
  });
  bool landed = true;
  for (const auto& b : bar) landed = landed && b.done == b.armed;
  if (!landed && (all || polls != 65u * slots)) return 1;              // gave up before the limit
  if (landed && open == static_cast<uint32_t>(slots) && at > static_cast<uint32_t>(slots) && !all) return 2;
  return polls <= 65u * slots ? 0 : 3;
}
}
