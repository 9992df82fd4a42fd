"""What the tiles of the plain GEMM cost beside their contraction, and what the walk makes of it."""
import shutil
import subprocess

import pytest

import test_tile_walk_cpu as walk

SOURCE = r"""
#include <cstdio>
#include <vector>
#include "%s"
using namespace msb;
// Last end in k-blocks, when a long tile takes k0 and a short one `cost`, with the rounds of `least`.
static long last(int n, int n0, int k0, int n1, int k1, long cost, long least) {
  const int rounds = least < 0 ? 0 : (int)walk_rounds(n0, k0, n1, walk_blocks(k1, least), n);
  long end = 0;
  for (int c = 0; c < n; ++c) {
    long work = 0;
    for (TileWalk w(c, n, n0, n0 + n1, rounds); w.more(); w.next()) work += w.t < n0 ? k0 : cost;
    end = work > end ? work : end;
  }
  return end;
}
int main() {
  // gradients of linear layers, tiles of 256 x 256: long ones, their k-blocks, short ones, theirs
  const int cases[][4] = {{54, 110, 504, 10}, {60, 121, 930, 7}, {72, 110, 504, 16}, {138, 123, 1426, 12}, {64, 64, 1024, 1}};
  for (const auto& c : cases) {
    // added to fp32 a short tile takes as long as 24 k-blocks, whatever its contraction: no pair ends later for the rounds
    if (last(74, c[0], c[1], c[2], c[3], 24, kWalkAdded32) > last(74, c[0], c[1], c[2], c[3], 24, -1)) printf("fp32: %%d tiles of %%d\n", c[0], c[1]);
    if (last(74, c[0], c[1], c[2], c[3], 48, kWalkAdded16) > last(74, c[0], c[1], c[2], c[3], 48, -1)) printf("bf16: %%d tiles of %%d\n", c[0], c[1]);
  }
  if (last(74, 54, 110, 504, 10, 24, 8) <= last(74, 54, 110, 504, 10, 24, kWalkAdded32)) printf("the rule does not see what it is for\n");
  // tiles of 128 or 256 columns: tokens, inputs, outputs, width of the gradients stored, and added to bf16 (each the faster one as measured)
  const int widths[][5] = {{2848, 2720, 472, 256, 128}, {1208, 1256, 2400, 256, 128}, {64, 16384, 4096, 256, 256}, {480, 272, 632, 128, 128}, {5400, 7344, 856, 256, 256}};
  for (const auto& w : widths)
    for (int adds = 0; adds < 2; ++adds) {
      WalkProblem p[2] = {{w[1], w[2], (w[0] + 63) / 64, adds != 0}, {w[0], w[1], (w[2] + 63) / 64, false}};
      if (p[1].kblocks > p[0].kblocks) { const WalkProblem t = p[0]; p[0] = p[1]; p[1] = t; }
      if (walk_tile_n(p, 2, 74) != w[3 + adds]) printf("%%d x %%d x %%d: %%d columns\n", w[0], w[1], w[2], walk_tile_n(p, 2, 74));
    }
  printf("done\n");
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_rounds_of_tiles_that_are_added_end_no_later_and_widths(tmp_path):
    src = tmp_path / "costs.cc"
    src.write_text(SOURCE % walk.HEADER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(tmp_path / "costs"), str(src)], check=True)
    r = subprocess.run([str(tmp_path / "costs")], capture_output=True, text=True)
    assert r.stdout == "done\n", r.stdout
