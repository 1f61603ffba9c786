"""CPU test of the phases that a reader waits for when it gives up in the middle of its ring."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "fa_ring.h"
#include <cstdio>

// Tile t goes into place t % S, in round t / S, whose phase has that number's parity.  The first S are asked for in advance, then one
// more for each that was read.  A reader that stops at tile x leaves the tiles from x on under way: are those the phases it waits for?
int main() {
  int wrong = 0, all = 0;
  for (int S = 1; S <= 8; ++S)
    for (int tiles = 1; tiles <= 5 * S; ++tiles) {
      int place = 0;
      unsigned phase = 0;
      for (int x = 0; x < tiles; ++x) {
        for (int t = x; t < tiles && t < x + S; ++t, ++all)
          wrong += fa::ring_phase(t % S, place, phase) != (static_cast<unsigned>(t / S) & 1u);
        if (++place == S) place = 0, phase ^= 1;
      }
    }
  std::printf("%d of %d", wrong, all);
  return wrong != 0 || all == 0;
}
"""


def test_copies_under_way_are_waited_for_in_their_own_phase(tmp_path):
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-I", os.path.join(ROOT, "triton_flashattn_b200", "csrc"), str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
