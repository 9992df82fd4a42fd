// A lane's 32 columns of a row of the result, in any layout of it.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace msb {

// out[at + i * step], i < n, of fp32 or bf16; whole vectors where they lie side by side on a 16-byte boundary.
__device__ __forceinline__ void store_row32(void* out, int64_t at, int64_t step, int n, bool fp32, const float (&v)[32]) {
  if (fp32) {
    float* o = reinterpret_cast<float*>(out) + at;
    if (n == 32 && step == 1 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<float4*>(o)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < n) o[i * step] = v[i];
    }
    return;
  }
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out) + at;
  if (n == 32 && step == 1 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * i + 2 * k], v[8 * i + 2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&b);
      }
      reinterpret_cast<uint4*>(o)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) o[i * step] = __float2bfloat16_rn(v[i]);
  }
}

}  // namespace msb
