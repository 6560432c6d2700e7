"""How many CTAs share the selection of an eviction, compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SWEEP = r"""
#include <cstdio>
#include <initializer_list>
#include "evict_plan.h"
using namespace tyr;
int main() {
  const int segment = 16384;
  long long bad = 0, n = 0;
  for (int places = 0; places < 16; ++places) {     // bit k - 1: the device can place a cluster of 2^k CTAs
    auto capacity = [&](int k) {
      if (k < 1 || k > 4) ++bad;
      return (places >> (k - 1)) & 1 ? 7 : 0;
    };
    for (long long x : {1ll, 2000ll, 16383ll, 16384ll, 16385ll, 32768ll, 32769ll, 65536ll, 65537ll, 131072ll, 131073ll, 262144ll, 262145ll, 1ll << 30}) {
      const int ranks = evict_ranks(x, segment, capacity);
      int k = 0;
      while (k < 4 && ((long long)segment << k) < x) ++k;
      const bool fits = ((long long)segment << k) >= x, placed = k == 0 || ((places >> (k - 1)) & 1);
      if (ranks != (fits && placed ? 1 << k : 1)) ++bad, std::printf("%lld keys, places %d: %d\n", x, places, ranks);
      ++n;
    }
  }
  int asked = 0;
  evict_ranks(segment, segment, [&](int) { return ++asked; });       // nothing is asked of the device where one CTA is enough
  evict_ranks((16ll << 14) + 1, segment, [&](int) { return ++asked; });
  std::printf("%lld choices, %lld bad, asked %d\n", n, bad, asked);
  return bad != 0 || asked != 0;
}
"""


def test_choices(tmp_path):
    src, exe = tmp_path / "sweep.cpp", tmp_path / "sweep"
    src.write_text(SWEEP)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "tyr_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
