"""The launch shape of the per-token scores, walked on the host."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hippolm_b200", "csrc")

_WALK = r"""
#include <stdio.h>
#include "token_logprobs_launch.h"
int main() {
  const int sms = 148;
  for (long long rows = 1; rows < 200000; rows = rows < 6000 ? rows + 1 : rows * 3 / 2)
    for (int parts = 1; parts <= 8; parts *= 2)
      for (int segs = 1; segs <= 1024; segs = segs < 20 ? segs + 1 : segs * 2)
        for (int top = 0; top < 2; ++top) {
          const int w = hippo::logprob_warps(rows, parts, segs, sms, top);
          const bool power = w == 1 || w == 2 || w == 4 || w == 8;
          // no warp without a segment; a block of many rows has warps enough for its row, one of few rows fills the card as far as it goes
          const long long blocks = rows * parts;
          const bool idle = blocks * w * 2 <= 32ll * sms && w * 2 <= segs && w < 8;
          const bool busy = w > 2 && w / 2 * 10 >= segs + 10 && blocks * (w / 2) > 32ll * sms;
          if (!power || w > segs || idle || busy) { printf("%lld rows, %d parts, %d segments, %d: %d warps\n", rows, parts, segs, top, w); return 1; }
        }
  return 0;
}
"""


def test_warps_of_a_block(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(_WALK)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_the_launch_takes_its_warps_from_the_rule():
    text = open(os.path.join(CSRC, "token_logprobs.cu")).read()
    assert "const int threads = 32 * logprob_warps(a.rows, parts, segs, sms, a.top > 0);" in text
