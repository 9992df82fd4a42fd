// The gated product by itself, for projections that other kernels compute (a mesh of several devices).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

// h = act(g) u;  dg = dh u act'(g), du = dh act(g).  bf16, n elements (a multiple of 8) on 16-byte boundaries.  act 0: silu, 1: tanh-GeLU.
cudaError_t gated_act(const void* g, const void* u, void* h, int64_t n, int act, cudaStream_t stream);
cudaError_t gated_act_bwd(const void* dh, const void* g, const void* u, void* dg, void* du, int64_t n, int act, cudaStream_t stream);

}  // namespace msb
