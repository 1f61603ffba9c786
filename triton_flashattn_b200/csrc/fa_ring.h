// The places of a ring and their phases (plain C++, so that it can be tested on the host).
#pragma once

namespace fa {

// A reader is at `place` of its ring, in a round whose copies complete the phase of parity `phase`.  The copies under way into the
// places from there on are of this round; those before it have been read and refilled for the next one.
constexpr unsigned ring_phase(int i, int place, unsigned phase) { return i < place ? phase ^ 1u : phase; }

}  // namespace fa
