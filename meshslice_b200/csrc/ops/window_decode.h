// One token per sequence over a cache of fixed size: the first `sinks` positions and the last `window`.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

struct WindowDecodeArgs {
  const void* qkv;             // bf16 [batch, kv * (group + 2) * 128], row pitch ld: per key/value head [q_0 | .. | q_group-1 | k | v]
  int64_t ld;
  void *k, *v;                 // bf16 [batch, kv, sinks + window, 128], contiguous
  const int64_t* positions;    // [batch] of these tokens; negative: an idle sequence
  void* out;                   // bf16 [batch, kv * group * 128], contiguous
  int batch, kv, group, window, sinks;
  float scale;
  // unused up to kWindowDecodeCluster splits:
  float* parts;                // fp32 [batch * kv * passes * splits * 16 * 130], passes = ceil(group / 16)
  uint32_t* counters;          // [batch * kv * passes], zero before the first launch and after each
};
constexpr int kWindowDecodePart = 16 * 130;   // floats of a split
constexpr int kWindowDecodeCluster = 8;       // splits that are joined within a cluster: the largest that every GPU of this kind has room for
// Splits of a sequence's slots that a launch uses on a GPU of `sms` SMs: sizes of `parts`.
int window_decode_splits(int batch, int kv, int group, int slots, int sms);
// Position p lies in slot p below `sinks` and in slot sinks + (p - sinks) % window from there on, so that the first
// min(p + 1, sinks + window) slots are exactly what token p sees, itself included.  The tokens' k and v are stored in their slots,
// out = softmax(q k^T scale) v over those slots; idle sequences store nothing and get zeros.
cudaError_t window_decode(const WindowDecodeArgs& a, int splits, cudaStream_t stream);

}  // namespace msb
