// Distillation from a teacher's top logits: loss and gradient of rows of logits.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

// Per row, with z the student's logits, p = softmax(t / T) over the entries the teacher kept (id in [0, vocab), the others are no
// entries) and y the label (outside [0, vocab): no label):
//   loss = w (log sum exp z - z_y) + (1 - w) T^2 sum_k p_k (log p_k - log softmax(z / T) at id_k)
//   grad = scale ( w (softmax z - onehot y) + (1 - w) T (softmax(z / T) - p) )
// A term without a label or without entries is zero.  The second term of the loss is a Kullback-Leibler divergence where every id occurs once;
// entries that share an id count as an event each, which takes a constant of the teacher off the loss and leaves the gradient as it is.
struct DistillArgs {
  const void* logits;          // bf16 [rows, cols]: columns [col_offset, col_offset + cols) of the vocabulary, pitch ld
  void* grad;                  // bf16 [rows, cols], pitch ldg; may be the logits
  int64_t ld, ldg;
  const int64_t* ids;          // [rows, top]
  const void* values;          // [rows, top], fp32 or bf16
  int values_bf16;
  const int64_t* targets;      // [rows], or null: no labels
  int rows, cols, col_offset, vocab, top;
  float temperature, hard, scale;
  float* loss;                 // [rows]
  float* stats;                // [rows, 5]: max, sum exp(z - max), sum exp((z - max) / T), sum p z, z_y (0 where not in this slice)
};
constexpr int kDistillTop = 1024;      // most entries of a row

// Whole rows of at most distill_row_cols() columns before the padding, in one pass over memory.
int distill_row_cols();
cudaError_t distill_row(const DistillArgs& a, cudaStream_t stream);
// Slices of rows, or longer rows: the statistics of a slice; the gradient (and, with `loss`, the loss) from those of whole rows.
cudaError_t distill_partial(const DistillArgs& a, cudaStream_t stream);
cudaError_t distill_grad(const DistillArgs& a, cudaStream_t stream);

}  // namespace msb
