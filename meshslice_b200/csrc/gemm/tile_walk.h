// Which tiles a CTA pair works on (plain C++: that every tile is taken once is checked on the CPU).
#pragma once
#include <stdint.h>

#ifndef MSB_HD
#ifdef __CUDACC__
#define MSB_HD __host__ __device__ __forceinline__
#else
#define MSB_HD inline
#endif
#endif

namespace msb {

// The tiles of a CTA pair.  Those of the first problem go round the pairs; where they do not come out even, the pairs that had one fewer
// take `rounds` of the next problem's (shorter) tiles among themselves, and from there on all pairs in turn, the early ones first.  In
// every round the pairs work on neighbouring tiles.  2047 x 1032 x 30011 and 30011 x 1032 x 2047 (40 tiles of 469 k-blocks and 590
// of 32): 241 us without those rounds.
struct TileWalk {
  int t;            // the tile, among those of all problems
  int clusters, cluster, first, all, late, skip;
  MSB_HD TileWalk(int cluster_, int clusters_, int first_, int all_, int rounds)
      : clusters(clusters_), cluster(cluster_), first(first_), all(all_), late(first_ % clusters_) {
    skip = rounds * (clusters - late);
    t = cluster < first ? cluster : enter();
  }
  MSB_HD int common() const { return first + skip + (cluster >= late ? cluster - late : cluster - late + clusters); }
  MSB_HD int enter() const { return skip > 0 && cluster >= late ? first + cluster - late : common(); }
  MSB_HD bool more() const { return t < all; }
  MSB_HD void next() {
    if (t < first) {
      t += clusters;
      if (t >= first) t = enter();
    } else if (t < first + skip) {
      t += clusters - late;
      if (t >= first + skip) t = common();
    } else {
      t += clusters;
    }
  }
};
// What a tile of `k` k-blocks takes, in k-blocks: however short its contraction, its sums are read and stored meanwhile, which takes as long as 8, and
// as 48 where they are added to 16-bit values.  Without that, few pairs get nearly all short tiles.  Gradients of a head (tokens x inputs x
// vocabulary), us by k-blocks alone and with leasts of 6, 8, 12 and 16: 52 x 632 x 82320 317, 171, 165, 166, 169; 32 x 2112 x 49464 524, 221, 210,
// 216, 223; 500 x 1024 x 50264 183, 183, 183, 187, 195.  Of a gated block of 512 x 4096 x 10752, added to bf16, by k-blocks alone and with leasts of
// 12, 24, 36 and 48: 1123, 1118, 1050, 1017, 999.
// In the plain GEMM, with four epilogue warps, a tile that the copy engine adds to fp32 values takes a pair as long as 24: where fewer than half of the
// pairs take rounds of them, those end last with a least of 8.  Where more do, memory is what bounds them all, and the more of it happens while
// others are on long tiles, the better.  Gradients of linear layers (tokens x inputs x outputs; pairs that take rounds), us without rounds and with leasts
// of 8, 20, 24 and 28: 640 x 4440 x 6992 (20) 94, 109, 92, 91, 90; 408 x 7664 x 7728 (14) 141, 164, 148, 146, 144; 1000 x 4440 x 6992 (2) 111, 123, 115, 110,
// 110; 736 x 11688 x 7816 (10) 301, 323, 302, 301, 301; 512 x 4096 x 16384 (42) 176, 146, 160, 163, 166; 64 x 4096 x 16384 (58) 150, 140, 144, 145, 145.
// The products, with eight, stay with 8: 500 x 1024 x 50264 198 us, with 16 and 24 212 and 218.
constexpr int64_t kWalkStored = 8, kWalkAdded32 = 24, kWalkAdded16 = 48;
inline int64_t walk_blocks(int64_t k, int64_t least = kWalkStored) { return k < least ? least : k; }
// Those rounds, for `n0` tiles of `k0` k-blocks and `n1` of `k1`, and the k-blocks of the pair that ends last.
inline int64_t walk_rounds(int64_t n0, int64_t k0, int64_t n1, int64_t k1, int64_t clusters) {
  const int64_t late = n0 % clusters;
  if (late == 0 || k1 < 1) return 0;
  const int64_t fit = k0 / k1, there = n1 / (clusters - late);
  return fit < there ? fit : there;
}
inline int64_t walk_end(int64_t n0, int64_t k0, int64_t n1, int64_t k1, int64_t clusters) {
  const int64_t late = n0 % clusters, early = clusters - late, rounds = walk_rounds(n0, k0, n1, k1, clusters), rest = n1 - rounds * early;
  const int64_t base = n0 / clusters * k0, common = rest / clusters * k1, odd = rest % clusters;      // `odd` tiles are left: early pairs first
  const int64_t ends_early = base + rounds * k1 + common + (odd > 0 ? k1 : 0);
  const int64_t ends_late = late > 0 ? base + k0 + common + (odd > early ? k1 : 0) : 0;
  return ends_early > ends_late ? ends_early : ends_late;
}


// The tile width that ends sooner.  A 64-deep k-block takes about 390 cycles on 128 columns (the loads: 24 KiB
// a CTA) and 530 on 256 (the tensor pipe: 512), so a narrow tile counts three quarters of a wide one.
// 2048 x 1024 x 4096 (32 wide tiles): 26.5 us wide, 19.6 narrow; 1024 x 2048 x 1024 11.9 and 8.7; 2048 x 2048 x 2048 (64
// wide tiles, one wave against two): wide, 16.3 us.
// A tile whose sums are added to 16-bit values costs its epilogue at least, a narrow one half of it, two thirds in its own k-blocks: linear
// layers' gradients by k-blocks alone and like this 2848 x 2720 x 472 49 and 35 us, 1208 x 1256 x 2400 33 and 31, 64 x 4096 x 16384 233 and 216, 232 x 3696 x
// 6880 106 and 98, 16 x 1536 x 12944 83 and 88.  For sums that are stored or added to fp32 it does not tell: priced so, wide tiles were chosen for
// 64 x 4096 x 16384 added to fp32, 169 us instead of 145.
struct WalkProblem {
  int64_t M, N, kblocks;
  bool adds_16;
};
inline int64_t walk_end(const WalkProblem* p, int problems, int tile_n, int64_t clusters) {
  int64_t tiles[2] = {0, 0}, k[2] = {0, 0};
  for (int i = 0; i < problems; ++i) {
    tiles[i] = (p[i].M + 255) / 256 * ((p[i].N + tile_n - 1) / tile_n);
    k[i] = p[i].adds_16 ? walk_blocks(p[i].kblocks, tile_n == 128 ? kWalkAdded16 * 2 / 3 : kWalkAdded16) : p[i].kblocks;
  }
  return walk_end(tiles[0], k[0], tiles[1], k[1], clusters);
}
inline int walk_tile_n(const WalkProblem* p, int problems, int64_t clusters) {
  return 3 * walk_end(p, problems, 128, clusters) < 4 * walk_end(p, problems, 256, clusters) ? 128 : 256;
}

}  // namespace msb
