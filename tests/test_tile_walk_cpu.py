"""The order in which CTA pairs take the tiles of one or two problems: every tile once, the long ones first, and evenly."""
import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parent.parent / "meshslice_b200" / "csrc" / "gemm" / "tile_walk.h"
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "%s"
using namespace msb;
static void fail(const char* what, int n, int n0, int n1, int k0, int k1) {
  printf("%%s: %%d pairs, %%d tiles of %%d, %%d of %%d\n", what, n, n0, k0, n1, k1);
  exit(1);
}
int main() {
  unsigned seed = 1;
  const auto rnd = [&](int m) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) %% (unsigned)m); };
  for (int trial = 0; trial < 20000; ++trial) {
    const int n = trial %% 3 ? 1 + rnd(80) : 74, n0 = rnd(300), n1 = trial %% 4 ? rnd(900) : 0, k0 = 1 + rnd(500), k1 = 1 + rnd(k0);
    const int rounds = (int)walk_rounds(n0, k0, n1, k1, n);
    std::vector<int> seen(n0 + n1, 0);
    long end = 0;
    for (int c = 0; c < n; ++c) {
      long work = 0;
      bool second = false;
      for (TileWalk w(c, n, n0, n0 + n1, rounds); w.more(); w.next()) {
        if (w.t < 0 || w.t >= n0 + n1 || seen[w.t]++) fail("a tile twice or none", n, n0, n1, k0, k1);
        if (w.t < n0 && second) fail("a long tile after a short one", n, n0, n1, k0, k1);
        second = second || w.t >= n0;
        work += w.t < n0 ? k0 : k1;
      }
      end = work > end ? work : end;
    }
    for (int s : seen) if (s != 1) fail("a tile is left", n, n0, n1, k0, k1);
    if (end != walk_end(n0, k0, n1, k1, n)) fail("another end than foreseen", n, n0, n1, k0, k1);
    // what no order can beat, and a short tile and the unevenness of the long ones that no short ones fill
    const long all = ((long)n0 * k0 + (long)n1 * k1 + n - 1) / n, longest = (long)((n0 + n - 1) / n) * k0;
    if (end > (all > longest ? all : longest) + 2 * k1) fail("uneven", n, n0, n1, k0, k1);
  }
  // a long contraction's tiles on all pairs but a few, and thousands of one k-block: those few do not get nearly all of them
  for (int late = 1; late < 74; ++late) {
    const int n = 74, n1 = 3483, rounds = (int)walk_rounds(late, walk_blocks(194), n1, walk_blocks(1), n);
    int most = 0;
    for (int c = 0; c < n; ++c) {
      int tiles = 0;
      for (TileWalk w(c, n, late, late + n1, rounds); w.more(); w.next()) tiles += w.t >= late;
      most = tiles > most ? tiles : most;
    }
    if (most > (n1 + n - 1) / n + 194 / 8 + 1) fail("short tiles on few pairs", n, late, n1, 194, 1);
  }
  printf("ok\n");
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_every_tile_once_and_evenly(tmp_path):
    src = tmp_path / "walk.cc"
    src.write_text(SOURCE % HEADER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(tmp_path / "walk"), str(src)], check=True)
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
