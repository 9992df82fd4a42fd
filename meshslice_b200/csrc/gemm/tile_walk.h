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
// What a tile of `k` k-blocks takes, in k-blocks: however short its contraction, its sums are read and stored, which took 2.4 us for
// 256 x 128 of them, as long as 12 k-blocks.  The gradients of 52 tokens, 632 inputs and 82320 columns, and of 32, 2112 and 49461, with a
// least of 6, 12 and 24: 174, 168 and 174 us, 223, 217 and 231 us; with none 318 and 530, for a few pairs then get nearly all short tiles.
inline int64_t walk_blocks(int64_t k) { return k < 12 ? 12 : k; }
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

}  // namespace msb
