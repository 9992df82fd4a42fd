// Rows of the head's loss, from what the product's epilogue wrote of each tile (gemm/sm100_products.h, kHead).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

// With z the logits of a row, m_t and s_t the maximum and the sum of exp(z - m_t) of tile t:
//   loss = log sum_t s_t exp(m_t - max m) + max m - z_y
//   p    = scale (softmax(z) - onehot y), bf16, over the exponentials e = exp(z - m_t) (fp16) that it replaces
// A row without a label (outside [0, vocab)) has loss 0 and p 0.
struct HeadRows {
  void* e;                   // fp16 in, bf16 out: [rows, cols], pitch ld; null: losses alone
  int64_t ld;
  const float2* stats;       // [tiles, rows]: m_t, s_t
  const float* label;        // [rows]: z_y
  const int64_t* targets;    // [rows]
  int rows, cols, tiles, tile_n, vocab;
  float scale;
  float* loss;               // [rows]
};
cudaError_t head_rows(const HeadRows& a, cudaStream_t stream);
// out [rows, cols] (bf16, cols a multiple of 4) = scale times the sum of `parts` fp32 matrices, `stride` elements apart, in their order.
cudaError_t sum_parts(const float* parts, int64_t stride, int n, void* out, int64_t rows, int64_t cols, float scale, cudaStream_t stream);

}  // namespace msb
