// Products of a few tokens with weights that are read once: the gated block's forward pass for single tokens.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

// Beyond them tiles of the tcgen05 pipe are faster.  Us here and there, weights [K, N]: 16 tokens of 1024 x 2816 22 and 28, of 4096 x 10752 81 and
// 89, of 8192 x 28672 300 and 288.
constexpr int kFewTokens = 16;

// out [tokens, N] = x W, or act(x W) * (x U) with `up`.  bf16, sums in fp32.  nt: the weights lie as [N, K], otherwise as [K, N]; rows begin on
// 16-byte boundaries, K and N are multiples of 8, tokens at most kFewTokens.
struct FewTokens {
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  const void* up;      // null: a plain product
  int64_t ldu;
  void* out;
  int64_t ldo;
  int tokens, K, N;
  int nt, act;
};
cudaError_t few_tokens(const FewTokens& a, cudaStream_t stream);

}  // namespace msb
