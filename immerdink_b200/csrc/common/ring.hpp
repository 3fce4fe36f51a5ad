// The end of a ring of copies after a wait that gave up: which phases are still to complete, and a bounded wait for
// them. Host + device, so that a host program can run it against a model of a barrier (tests/ring_shim.cpp).
#pragma once
#include "wide.hpp"

namespace imd {

// Loads go to slots 0, 1, ..., slots - 1, 0, ... and each arms its slot's barrier for one phase. Parity of the phase that
// slot s was armed for last, of the first `issued` loads; -1 for a slot that none of them used. A barrier answers a
// question for the other parity at once (the phase before has completed), so only this one says whether the copy landed.
IMD_HD int last_parity(uint32_t issued, int slots, int s) {
  return issued <= static_cast<uint32_t>(s) ? -1 : static_cast<int>((issued - 1 - s) / slots & 1u);
}

// Polls until the last copy of every slot has landed, at most `limit` times each. try_wait(s, parity): whether the phase of
// that parity of slot s's barrier has completed. Returns whether all have.
template <typename TryWait>
IMD_HD bool await_ring(uint32_t issued, int slots, uint32_t limit, TryWait try_wait) {
  for (uint32_t it = 0; it < limit; ++it) {
    bool landed = true;
    for (int s = 0; s < slots; ++s) {
      const int parity = last_parity(issued, slots, s);
      if (parity >= 0 && !try_wait(s, static_cast<uint32_t>(parity))) landed = false;
    }
    if (landed) return true;
  }
  return false;
}

// The same without the number of loads: until the phase that each slot is in now has completed. A slot that waits for no
// copy takes all of the limit. At most 32 slots.
template <typename TryWait>
IMD_HD bool await_slots(int slots, uint32_t limit, TryWait try_wait) {
  uint32_t now = 0;  // bit s: the parity of slot s's phase; the other's has completed
  for (int s = 0; s < slots; ++s) now |= (try_wait(s, 0u) ? 1u : 0u) << s;
  for (uint32_t it = 0; it < limit; ++it) {
    bool landed = true;
    for (int s = 0; s < slots; ++s)
      if (!try_wait(s, now >> s & 1u)) landed = false;
    if (landed) return true;
  }
  return false;
}

}  // namespace imd
