#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "../common/pdl.cuh"
#include "head.h"

namespace msb {

namespace {

constexpr int kThreads = 256;

template <class F>
__device__ __forceinline__ float block_join(float v, float* red, F join) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v = join(v, red[i]);
  __syncthreads();
  return v;
}

}  // namespace

// A CTA per row: joins the tiles' statistics, then turns the exponentials into the gradient in place, 16 bytes a thread.  HBM bounds it:
// 4 bytes an element.
__global__ void __launch_bounds__(kThreads)
head_rows_kernel(const HeadRows a) {
  grid_trigger();
  grid_wait();
  extern __shared__ float factor[];        // [tiles]: scale exp(m_t - max m) / sum
  __shared__ float red[kThreads / 32];
  const int row = blockIdx.x;
  const int64_t y = a.targets[row];
  const bool label = y >= 0 && y < a.vocab;
  float m = -CUDART_INF_F;
  for (int t = threadIdx.x; t < a.tiles; t += kThreads) m = fmaxf(m, a.stats[(int64_t)t * a.rows + row].x);
  const float top = block_join(m, red, [](float x, float w) { return fmaxf(x, w); });
  float s = 0.f;
  for (int t = threadIdx.x; t < a.tiles; t += kThreads) {
    const float2 st = a.stats[(int64_t)t * a.rows + row];
    // a tile with nothing above -inf adds nothing, unless it held a NaN
    if (st.y != 0.f) s += st.y * expf(st.x - top);
  }
  const float total = block_join(s, red, [](float x, float w) { return x + w; });
  float zy = 0.f;
  if (threadIdx.x == 0 || a.e != nullptr) zy = label ? a.label[row] : 0.f;
  if (threadIdx.x == 0) a.loss[row] = label ? logf(total) + (top - zy) : 0.f;
  if (a.e == nullptr) return;
  uint4* const e = reinterpret_cast<uint4*>(reinterpret_cast<__half*>(a.e) + row * a.ld);
  if (!label) {
    for (int i = threadIdx.x; i < a.cols / 8; i += kThreads) e[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const float over = a.scale / total;
  for (int t = threadIdx.x; t < a.tiles; t += kThreads) {
    const float2 st = a.stats[(int64_t)t * a.rows + row];
    factor[t] = st.y != 0.f ? over * expf(st.x - top) : 0.f;
  }
  __syncthreads();
  const int at_y = (int)(y >> 3);
  for (int i = threadIdx.x; i < a.cols / 8; i += kThreads) {
    const float f = factor[i * 8 / a.tile_n];
    uint4 v = e[i];
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      const __nv_bfloat162 o = __floats2bfloat162_rn(x.x * f, x.y * f);
      w[j] = *reinterpret_cast<const uint32_t*>(&o);
    }
    if (i == at_y) {      // from the label's logit in fp32: the difference to 1 is rounded once
      const __nv_bfloat16 d = __float2bfloat16_rn(a.scale * (expf(zy - top) / total - 1.f));
      const int j = (int)y & 7;
      const uint32_t bits = (uint32_t)__bfloat16_as_ushort(d);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j >> 1 == k) w[k] = j & 1 ? (w[k] & 0xffffu) | bits << 16 : (w[k] & 0xffff0000u) | bits;
    }
    e[i] = v;
  }
}

cudaError_t head_rows(const HeadRows& a, cudaStream_t stream) {
  if (a.cols % 8 || a.ld % 8 || a.tile_n % 8 || a.tiles > 8192) return cudaErrorInvalidValue;
  return launch_dependent(head_rows_kernel, a.rows, kThreads, a.tiles * sizeof(float), stream, a);
}

}  // namespace msb
