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

// A CTA per row: joins the tiles' statistics, then turns the exponentials into the gradient in place, 16 bytes a thread and four of
// them in flight.  HBM bounds it: 4 bytes an element.
__global__ void __launch_bounds__(kThreads)
head_rows_kernel(const HeadRows a) {
  grid_trigger();
  grid_wait();
  extern __shared__ float2 joined[];       // [tiles]: m_t and s_t, then .x: scale exp(m_t - max m) / sum
  __shared__ float red[kThreads / 32];
  const int row = blockIdx.x;
  const int64_t y = a.targets[row];
  const bool label = y >= 0 && y < a.vocab;
  uint4* const e = reinterpret_cast<uint4*>(reinterpret_cast<__half*>(a.e) + row * a.ld);
  const int vectors = a.cols / 8;
  if (!label) {
    if (threadIdx.x == 0) a.loss[row] = 0.f;
    for (int i = threadIdx.x; i < vectors; i += kThreads) e[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const float zy = a.label[row];
  float m = -CUDART_INF_F;
  for (int t = threadIdx.x; t < a.tiles; t += kThreads) {
    const float2 st = a.stats[(int64_t)t * a.rows + row];
    joined[t] = st;
    m = fmaxf(m, st.x);
  }
  const float top = block_join(m, red, [](float x, float w) { return fmaxf(x, w); });
  float s = 0.f;
  for (int t = threadIdx.x; t < a.tiles; t += kThreads) {
    // a tile with nothing above -inf adds nothing, unless it held a NaN
    if (joined[t].y != 0.f) s += joined[t].y * expf(joined[t].x - top);
  }
  const float total = block_join(s, red, [](float x, float w) { return x + w; });
  if (threadIdx.x == 0) a.loss[row] = logf(total) + (top - zy);
  const float over = a.scale / total;
  for (int t = threadIdx.x; t < a.tiles; t += kThreads) joined[t].x = joined[t].y != 0.f ? over * expf(joined[t].x - top) : 0.f;
  __syncthreads();
  const int at_y = (int)(y >> 3), per = a.tile_n / 8;
  constexpr int kFlight = 4;
  for (int i0 = threadIdx.x; i0 < vectors; i0 += kFlight * kThreads) {
    uint4 v[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i0 + k * kThreads < vectors) v[k] = e[i0 + k * kThreads];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int i = i0 + k * kThreads;
      if (i >= vectors) break;
      const float f = joined[i / per].x;
      uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
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
        for (int q = 0; q < 4; ++q)
          if (j >> 1 == q) w[q] = j & 1 ? (w[q] & 0xffffu) | bits << 16 : (w[q] & 0xffff0000u) | bits;
      }
      e[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// Losses alone: a lane per row, so that the statistics of neighbouring rows are read together, and the tiles shared out to the warps of a
// CTA, each of which keeps a running maximum and sum.
constexpr int kLossWarps = 16;
__global__ void __launch_bounds__(32 * kLossWarps)
head_losses_kernel(const HeadRows a) {
  grid_trigger();
  grid_wait();
  __shared__ float2 part[kLossWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 32 + lane;
  float m = -CUDART_INF_F, s = 0.f;
  const auto take = [&](float2 st) {
    if (st.y == 0.f) return;                     // nothing above -inf
    const float top = fmaxf(m, st.x);
    s = (m == -CUDART_INF_F ? 0.f : s * expf(m - top)) + st.y * expf(st.x - top);
    m = top;
  };
  if (row < a.rows) {
    constexpr int kFlight = 4;
    for (int t0 = warp; t0 < a.tiles; t0 += kFlight * kLossWarps) {
      float2 st[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k)
        st[k] = t0 + k * kLossWarps < a.tiles ? a.stats[(int64_t)(t0 + k * kLossWarps) * a.rows + row] : make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kFlight; ++k) take(st[k]);
    }
  }
  part[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (warp != 0 || row >= a.rows) return;
  m = -CUDART_INF_F;
  s = 0.f;
  for (int k = 0; k < kLossWarps; ++k) take(part[k][lane]);
  const int64_t y = a.targets[row];
  a.loss[row] = y >= 0 && y < a.vocab ? logf(s) + (m - a.label[row]) : 0.f;
}

__global__ void __launch_bounds__(kThreads)
sum_parts_kernel(const float* parts, int64_t stride, int n, uint2* out, int64_t vectors, float scale) {
  grid_trigger();
  grid_wait();
  const int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (i >= vectors) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const float4 v = reinterpret_cast<const float4*>(parts + k * stride)[i];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  const __nv_bfloat162 lo = __floats2bfloat162_rn(s.x * scale, s.y * scale), hi = __floats2bfloat162_rn(s.z * scale, s.w * scale);
  out[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

cudaError_t sum_parts(const float* parts, int64_t stride, int n, void* out, int64_t rows, int64_t cols, float scale, cudaStream_t stream) {
  const int64_t vectors = rows * cols / 4;
  if (cols % 4 || stride % 4 || vectors > (int64_t)1 << 38) return cudaErrorInvalidValue;
  return launch_dependent(sum_parts_kernel, (unsigned)((vectors + kThreads - 1) / kThreads), kThreads, 0, stream, parts, stride, n,
                          reinterpret_cast<uint2*>(out), vectors, scale);
}
cudaError_t head_rows(const HeadRows& a, cudaStream_t stream) {
  if (a.e == nullptr) return launch_dependent(head_losses_kernel, (a.rows + 31) / 32, 32 * kLossWarps, 0, stream, a);
  if (a.cols % 8 || a.ld % 8 || a.tile_n % 8 || a.tiles > 4096) return cudaErrorInvalidValue;
  return launch_dependent(head_rows_kernel, a.rows, kThreads, a.tiles * sizeof(float2), stream, a);
}

}  // namespace msb
