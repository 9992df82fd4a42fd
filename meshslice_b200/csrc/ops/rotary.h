// Rotary positions on rows of grouped heads: per key/value head [q_0 | .. | q_group-1 | k | v], head_dim features each.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

struct RotaryArgs {
  const void* x;               // bf16 [tokens, kv * (group + 2) * head_dim], row pitch ldx elements
  void* y;                     // the same with row pitch ldy, or x itself
  int64_t ldx, ldy;
  const int64_t* positions;    // [tokens], or null: token % seq
  const uint64_t* turns;       // [rot_dim / 2] turns per position, in units of 2^-64
  int tokens, seq, kv, group, head_dim, rot_dim;
  int half;                    // pairs are (i, i + rot_dim / 2); otherwise (2 i, 2 i + 1)
  float sign, factor;          // of the angle; of cosine and sine
};

// The first rot_dim features of every query and key head are rotated by position * turns, the others and the value heads copied
// (left alone where y is x).  head_dim and rot_dim are multiples of 16, rows 16-byte aligned (cudaErrorInvalidValue otherwise).
cudaError_t rotary(const RotaryArgs& a, cudaStream_t stream);

}  // namespace msb
