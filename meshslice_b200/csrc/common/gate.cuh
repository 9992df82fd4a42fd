// Activations of gated feed-forward blocks in fp32.  Both are x sigmoid(q(x)): q(x) = x (silu), 2 sqrt(2 / pi) (x + 0.044715 x^3) (tanh-GeLU, since
// 1 + tanh(y) = 2 sigmoid(2 y)), with ex2.approx and a division of 2 units in the last place.  A value is off by at most (8 |q| + 16) 2^-24 of it
// where q is negative: the roundings of q, up to six, and of its product with log2 e are shares of the exponential there.  That is 2^-20 near 0, 2^-17.5
// for a GeLU of -4 (q = -11), 2^-14 where the sigmoid leaves fp32 (q = -87), all far below the 2^-9 of a result in bf16; where q is positive 2^-20.
// tanh.approx would leave 2^-11 everywhere.
#pragma once
#include <cuda_runtime.h>

namespace msb {

// act 0: silu, 1: GeLU.  sigmoid(q(x))
__device__ __forceinline__ float gate_sigmoid(float x, int act) {
  const float q = act == 0 ? x : 1.5957691216057308f * (x + 0.044715f * x * x * x);
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * q));
  return __fdividef(1.f, 1.f + e);
}
// The activation's derivative, with s = sigmoid(q(x)).
__device__ __forceinline__ float gate_slope(float x, float s, int act) {
  const float c = fminf(fabsf(x), 64.f);       // beyond, s is 0 or 1 and 1 - s or s without a rest, and x x may leave fp32: 0 times infinity
  const float dq = act == 0 ? 1.f : 1.5957691216057308f * (1.f + 3.f * 0.044715f * c * c);
  return s + x * s * (1.f - s) * dq;
}

}  // namespace msb
