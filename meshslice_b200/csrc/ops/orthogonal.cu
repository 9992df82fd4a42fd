#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../common/pdl.cuh"
#include "orthogonal.h"

namespace msb {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float element(const void* g, int bf16, int64_t i) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(g)[i]) : reinterpret_cast<const float*>(g)[i];
}

}  // namespace

// In 64 bits: squares of gradients leave the range of fp32 (1e-23), and the order of the parts is fixed.
__global__ void __launch_bounds__(kThreads)
square_sums_kernel(const void* g, int bf16, int64_t items, int64_t n, int64_t stride, int64_t per, double* partial) {
  grid_trigger();
  grid_wait();
  __shared__ double red[kThreads / 32];
  for (int64_t item = blockIdx.y; item < items; item += gridDim.y) {
    const int64_t first = item * stride + blockIdx.x * per, last = item * stride + min(n, (int64_t)(blockIdx.x + 1) * per);
    double s = 0.0;
    int64_t i = first + threadIdx.x;
    for (; i + 3 * kThreads < last; i += 4 * kThreads) {      // four loads in flight
      const float v0 = element(g, bf16, i), v1 = element(g, bf16, i + kThreads), v2 = element(g, bf16, i + 2 * kThreads),
                  v3 = element(g, bf16, i + 3 * kThreads);
      s += ((double)v0 * v0 + (double)v1 * v1) + ((double)v2 * v2 + (double)v3 * v3);
    }
    for (; i < last; i += kThreads) {
      const double v = element(g, bf16, i);
      s += v * v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < kThreads / 32; ++k) s += red[k];
      partial[item * kNormParts + blockIdx.x] = s;
    }
    __syncthreads();
  }
}

// Tiles of 32 x 32, through shared memory where the matrix is transposed.
__global__ void __launch_bounds__(kThreads)
load_unit_kernel(const LoadUnit a) {
  grid_trigger();
  grid_wait();
  __shared__ float tile[32][33];
  __shared__ double inverse;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int item = blockIdx.z; item < a.items; item += gridDim.z) {
    if (threadIdx.x < 32) {
      double s = 0.0;
      for (int k = threadIdx.x; k < a.parts; k += 32) s += a.partial[(int64_t)item * kNormParts + k];
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (threadIdx.x == 0) inverse = s == 0.0 ? 0.0 : 1.0 / sqrt(s);
    }
    __syncthreads();
    const double inv = inverse;
    for (int r0 = blockIdx.y * 32; r0 < a.mp; r0 += gridDim.y * 32) {
      const int c0 = blockIdx.x * 32;
      const int64_t out0 = ((int64_t)item * a.mp + r0) * a.np + c0;
      if (a.transpose) {
#pragma unroll
        for (int k = 0; k < 32; k += kThreads / 32) {      // G's rows are X's columns
          const int r = c0 + ty + k, c = r0 + tx;
          tile[ty + k][tx] = r < a.rows && c < a.cols ? element(a.g, a.bf16, item * a.stride + (int64_t)r * a.cols + c) : 0.f;
        }
        __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < 32; k += kThreads / 32) {
        const int r = r0 + ty + k, c = c0 + tx;
        float v;
        if (a.transpose) v = tile[tx][ty + k];
        else v = r < a.rows && c < a.cols ? element(a.g, a.bf16, item * a.stride + (int64_t)r * a.cols + c) : 0.f;
        const float x = (float)((double)v * inv);
        const int64_t at = out0 + (int64_t)(ty + k) * a.np + tx;
        a.x[at] = x;
        reinterpret_cast<__half*>(a.xs)[at] = __float2half_rn(x * a.scale);
      }
      if (a.transpose) __syncthreads();
    }
    __syncthreads();
  }
}

// Four elements a thread; HBM bounds both: 16 bytes an element (12 with gradients in 16 bits) and 14.
__global__ void __launch_bounds__(kThreads)
momentum_kernel(const void* grad, int grad_fp32, float4* m, float4* u, int64_t items, int64_t nvec, int64_t stride, float momentum,
                int nesterov, const float* grad_scale) {
  grid_trigger();
  grid_wait();
  const float s = grad_scale != nullptr ? *grad_scale : 1.f;
  for (int64_t item = blockIdx.y; item < items; item += gridDim.y)
    for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < nvec; i += (int64_t)gridDim.x * kThreads) {
      const int64_t at = item * stride + i;
      float4 g;
      if (grad_fp32) {
        g = reinterpret_cast<const float4*>(grad)[at];
      } else {
        const uint2 w = reinterpret_cast<const uint2*>(grad)[at];
        g = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                        __uint_as_float(w.y & 0xffff0000u));
      }
      float4 v = m[at];
      g.x *= s; g.y *= s; g.z *= s; g.w *= s;
      v.x = momentum * v.x + g.x;
      v.y = momentum * v.y + g.y;
      v.z = momentum * v.z + g.z;
      v.w = momentum * v.w + g.w;
      m[at] = v;
      if (nesterov) v = make_float4(g.x + momentum * v.x, g.y + momentum * v.y, g.z + momentum * v.z, g.w + momentum * v.w);
      u[item * nvec + i] = v;
    }
}
__global__ void __launch_bounds__(kThreads)
apply_update_kernel(const float4* o, float4* master, uint2* param, int64_t items, int64_t nvec, int64_t stride, float lr, float size,
                    float wd) {
  grid_trigger();
  grid_wait();
  for (int64_t item = blockIdx.y; item < items; item += gridDim.y)
    for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < nvec; i += (int64_t)gridDim.x * kThreads) {
      const int64_t at = item * stride + i;
      const float4 d = o[item * nvec + i];
      float4 w = master[at];
      w.x -= lr * (size * d.x + wd * w.x);
      w.y -= lr * (size * d.y + wd * w.y);
      w.z -= lr * (size * d.z + wd * w.z);
      w.w -= lr * (size * d.w + wd * w.w);
      master[at] = w;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(w.x, w.y), hi = __floats2bfloat162_rn(w.z, w.w);
      param[at] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
}

static dim3 flat_grid(int64_t items, int64_t nvec) {
  const int64_t want = (nvec + kThreads - 1) / kThreads;
  return dim3((unsigned)(want < (1 << 22) ? want : 1 << 22), (unsigned)(items < 4096 ? items : 4096));
}
cudaError_t momentum_step(const void* grad, int grad_fp32, float* m, float* u, int64_t items, int64_t n, int64_t stride, float momentum,
                          int nesterov, const float* grad_scale, cudaStream_t stream) {
  if (n % 4 || (items > 1 && stride % 4)) return cudaErrorInvalidValue;
  return launch_dependent(momentum_kernel, flat_grid(items, n / 4), kThreads, 0, stream, grad, grad_fp32, reinterpret_cast<float4*>(m),
                          reinterpret_cast<float4*>(u), items, n / 4, stride / 4, momentum, nesterov, grad_scale);
}
cudaError_t apply_update(const float* o, float* master, void* param, int64_t items, int64_t n, int64_t stride, float lr, float size, float wd,
                         cudaStream_t stream) {
  if (n % 4 || (items > 1 && stride % 4)) return cudaErrorInvalidValue;
  return launch_dependent(apply_update_kernel, flat_grid(items, n / 4), kThreads, 0, stream, reinterpret_cast<const float4*>(o),
                          reinterpret_cast<float4*>(master), reinterpret_cast<uint2*>(param), items, n / 4, stride / 4, lr, size, wd);
}

int norm_parts(int64_t n) {
  const int64_t want = (n + 8191) / 8192;
  return (int)(want < 1 ? 1 : want > kNormParts ? kNormParts : want);
}
cudaError_t square_sums(const void* g, int bf16, int64_t items, int64_t n, int64_t stride, double* partial, cudaStream_t stream) {
  const int parts = norm_parts(n);
  const int64_t per = (n + parts - 1) / parts;
  return launch_dependent(square_sums_kernel, dim3(parts, (unsigned)(items < 4096 ? items : 4096)), kThreads, 0, stream, g, bf16, items, n,
                          stride, per, partial);
}
cudaError_t load_unit(const LoadUnit& a, cudaStream_t stream) {
  if (a.mp % 32 || a.np % 32 || a.parts > kNormParts) return cudaErrorInvalidValue;
  const int rows = a.mp / 32 < 4096 ? a.mp / 32 : 4096;
  return launch_dependent(load_unit_kernel, dim3(a.np / 32, rows, (unsigned)(a.items < 4096 ? a.items : 4096)), kThreads, 0, stream, a);
}

}  // namespace msb
