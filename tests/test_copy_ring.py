"""How the cache attention's ring of copies is left when a wait runs out (nothing of it may still be under way when a block ends)."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hippolm_b200", "csrc")

# Copy c goes to stage c % S and completes phase c / S of that stage's barrier; a wait for a parity ends at once where the barrier is in a
# phase of the other parity. While copy c is under way its barrier is in phase c / S.
_WALK = r"""
#include <stdio.h>
#include "ring.h"
int main() {
  for (int S = 2; S <= 3; ++S)
    for (int tiles = 1; tiles <= 13; ++tiles) {
      int stage = 0, phase = 0;
      for (int i = 0; i < tiles; ++i) {                  // the wait for copy i runs out; copies up to `issued` are under way
        const int issued = i + S < tiles ? i + S : tiles;
        for (int c = i; c < issued; ++c) {
          const hippo::RingPlace r = hippo::ring_place(stage, phase, c - i, S);
          if (r.stage != c % S || r.parity != (c / S & 1)) { printf("S %d, copy %d of %d at %d\n", S, c, tiles, i); return 1; }
        }
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
    }
  return 0;
}
"""


def test_places_of_the_copies_under_way(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(_WALK)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_cache_attention_drains_the_places_of_its_copies():
    text = open(os.path.join(CSRC, "kv8_attention.cu")).read()
    drain = text[text.index("if (!alive)"):]
    drain = drain[:drain.index("found.x = -1")]
    # one wait for every tile between the next one to be used and the next one to be fetched, at its own place
    assert "get.left != put.left" in drain and "get.advance(a)" in drain
    assert re.search(r"ring_place\(stage, phase, \w+, S::kStages\)", drain)
    assert re.findall(r"mbar_wait\(&full\[([^\]]*)\], ([^,]*),", drain) == [("r.stage", "r.parity")]


def test_cache_attention_gives_up_as_a_whole_warp():
    """The lanes' waits run out one by one: the warp acts on their common result (its next shuffles name all lanes)."""
    text = open(os.path.join(CSRC, "kv8_attention.cu")).read()
    body = text[:text.index("if (!alive)")]
    waits = [line.strip() for line in body.splitlines() if "mbar_wait(" in line]
    assert waits and all(re.match(r"const bool (\w+) = mbar_wait\(.*\);", w) or "__all_sync(" in w for w in waits), waits
    for name in re.findall(r"const bool (\w+) = mbar_wait\(", body):
        assert re.search(rf"if \(!__all_sync\(0xffffffffu, {name}\)\)", body), name
