// What the orthogonal update of a matrix needs beside its products (gemm/sm100_products.h, kGram and kStep).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

constexpr int kNormParts = 256;      // most partial sums of a matrix
// Sums of squares of `items` matrices of `n` contiguous elements each (fp32 or bf16), `stride` elements apart: partial sums in 64 bits
// [items, kNormParts], norm_parts(n) of each.
int norm_parts(int64_t n);
// Clears `zeros` words at `clear` too.
cudaError_t square_sums(const void* g, int bf16, int64_t items, int64_t n, int64_t stride, double* partial, uint32_t* clear, int zeros,
                        cudaStream_t stream);
// X = G / |G| (0 where G is 0), or its transpose, padded with zeros to [mp, np]: fp32, and `scale` times it in fp16.
struct LoadUnit {
  const void* g;
  int bf16;
  int64_t stride;              // elements from one matrix to the next
  int items, rows, cols;       // of G
  int transpose;
  const double* partial;
  int parts;
  float* x;                    // [items, mp, np]
  void* xs;                    // fp16 [items, mp, np]
  int mp, np;
  float scale;
};
cudaError_t load_unit(const LoadUnit& a, cudaStream_t stream);

// All of it for matrices of up to kUnitSide rows and columns, in one launch.
constexpr int kUnitSide = 256;
constexpr uint32_t kUnitTimeout = 60;        // status: waited too long for a product
struct UnitSmall {
  const void* g;
  int bf16;
  int64_t stride;              // elements from one matrix to the next
  int items, rows, cols, steps;
  float a, b, c;
  void* out;
  int out_fp32;
  int64_t out_item, out_row, out_col;        // strides in elements
  uint32_t* status;
  uint64_t timeout_ns;
};
cudaError_t orthogonal_small(const UnitSmall& a, cudaStream_t stream);

// The optimizer step around it, on `items` matrices of n elements (a multiple of 4) that lie `stride` elements apart in the flat buffers:
//   m <- momentum m + s g,   u = s g + momentum m (nesterov) or m            s: *grad_scale, 1 for null
//   master <- master - lr (size o + wd master), param = bf16(master)         u, o: [items, n], fp32
cudaError_t momentum_step(const void* grad, int grad_fp32, float* m, float* u, int64_t items, int64_t n, int64_t stride, float momentum,
                          int nesterov, const float* grad_scale, cudaStream_t stream);
cudaError_t apply_update(const float* o, float* master, void* param, int64_t items, int64_t n, int64_t stride, float lr, float size, float wd,
                         cudaStream_t stream);

}  // namespace msb
