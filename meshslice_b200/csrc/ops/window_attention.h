// Causal attention within a window that keeps the first tokens visible: query i sees key j <= i where i - j < window or j < sinks.
// head_dim 128, bf16, on tcgen05.  qkv [batch * seq, kv * (group + 2) * 128], columns per key/value head
// [q_0 | .. | q_group-1 | k | v]; out / dout [batch * seq, kv * group * 128].  Any seq.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

struct WindowShape {
  int batch, seq, kv, group;
  int window;                  // 0: no window
  int sinks;
  float scale;
};

// out = softmax over what a query sees of (q k^T scale), times v; lse[b, head, s] = log sum exp of the scaled scores.
// qkv and out start on 16-byte boundaries (cudaErrorInvalidValue otherwise).  status: 4 words, first error wins.
cudaError_t window_attention_fwd(const void* qkv, void* out, float* lse, const WindowShape& s, uint32_t* status, cudaStream_t stream);

// dqkv from dout.  `scratch`: window_attention_scratch() fp32 values.  All tensors start on 16-byte boundaries.  Bit-identical from
// run to run.
int64_t window_attention_scratch(const WindowShape& s);
cudaError_t window_attention_bwd(const void* qkv, const void* out, const void* dout, const float* lse, void* dqkv, float* scratch,
                                 const WindowShape& s, uint32_t* status, cudaStream_t stream);

}  // namespace msb
