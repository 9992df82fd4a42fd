#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../common/pdl.cuh"
#include "orthogonal.h"

namespace msb {

namespace {

constexpr int kThreads = 256, kSumThreads = 512;

__device__ __forceinline__ float element(const void* g, int bf16, int64_t i) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(g)[i]) : reinterpret_cast<const float*>(g)[i];
}

}  // namespace

// In 64 bits: squares of gradients leave the range of fp32 (1e-23), and the order of the parts is fixed.  A thread has four vectors in
// flight: 4096 x 16384 in fp32 (268 MB) 300 us with four elements, in 128 parts.
__global__ void __launch_bounds__(kSumThreads)
square_sums_kernel(const void* g, int bf16, int64_t items, int64_t n, int64_t stride, int64_t per, double* partial, uint32_t* clear, int zeros) {
  grid_trigger();
  grid_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < zeros; i += kSumThreads) clear[i] = 0;
  __shared__ double red[kSumThreads / 32];
  const int wide = bf16 ? 8 : 4, bytes = bf16 ? 2 : 4;
  for (int64_t item = blockIdx.y; item < items; item += gridDim.y) {
    const int64_t first = (int64_t)blockIdx.x * per, last = min(n, first + per);          // `per` is a multiple of 8
    const char* const base = reinterpret_cast<const char*>(g) + item * stride * bytes;
    double s = 0.0;
    int64_t done = first;
    if ((reinterpret_cast<uintptr_t>(base) & 15) == 0 && last > first) {
      const int64_t vectors = (last - first) / wide;
      const uint4* const v = reinterpret_cast<const uint4*>(base + first * bytes);
      for (int64_t i = threadIdx.x; i < vectors; i += 4 * kSumThreads) {
        uint4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = i + k * kSumThreads < vectors ? v[i + k * kSumThreads] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (bf16) {
              const double a = __uint_as_float(w[j] << 16), b = __uint_as_float(w[j] & 0xffff0000u);
              s += a * a + b * b;
            } else {
              const double a = __uint_as_float(w[j]);
              s += a * a;
            }
          }
        }
      }
      done = first + vectors * wide;
    }
    for (int64_t i = done + threadIdx.x; i < last; i += kSumThreads) {
      const double a = element(base, bf16, i);
      s += a * a;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < kSumThreads / 32; ++k) s += red[k];
      partial[item * kNormParts + blockIdx.x] = s;
    }
    __syncthreads();
  }
}

// 1 / |G| of an item (0 for G = 0), to all threads.
__device__ __forceinline__ double inverse_norm(const double* partial, int parts, double* red) {
  double s = (int)threadIdx.x < parts ? partial[threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) s += red[k];
  return s == 0.0 ? 0.0 : 1.0 / sqrt(s);
}

// As G lies: four columns a thread.
__global__ void __launch_bounds__(kThreads)
load_unit_kernel(const LoadUnit a) {
  grid_trigger();
  grid_wait();
  __shared__ double red[kThreads / 32];
  const int groups = a.np / 4;
  const bool whole = a.cols % 4 == 0 && a.stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.g) & 15) == 0;
  for (int item = blockIdx.y; item < a.items; item += gridDim.y) {
    const double inv = inverse_norm(a.partial + (int64_t)item * kNormParts, a.parts, red);
    for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < (int64_t)a.mp * groups; i += (int64_t)gridDim.x * kThreads) {
      const int r = (int)(i / groups), c = (int)(i - (int64_t)r * groups) * 4;
      const int64_t from = item * a.stride + (int64_t)r * a.cols + c;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < a.rows && c < a.cols) {
        if (whole && !a.bf16) {
          const float4 t = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.g) + from);
          v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else if (whole) {
          const uint2 t = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(a.g) + from);
          v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
          v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c + k < a.cols) v[k] = element(a.g, a.bf16, from + k);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = (float)((double)v[k] * inv);
      const int64_t at = (int64_t)item * a.mp * a.np + i * 4;
      *reinterpret_cast<float4*>(a.x + at) = make_float4(v[0], v[1], v[2], v[3]);
      const __half2 lo = __floats2half2_rn(v[0] * a.scale, v[1] * a.scale), hi = __floats2half2_rn(v[2] * a.scale, v[3] * a.scale);
      *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(a.xs) + at) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}

// Transposed, by way of shared memory: tiles of 32 x 32.
__global__ void __launch_bounds__(kThreads)
load_unit_transposed_kernel(const LoadUnit a) {
  grid_trigger();
  grid_wait();
  __shared__ float tile[32][33];
  __shared__ double red[kThreads / 32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = blockIdx.x * 32;
  for (int item = blockIdx.z; item < a.items; item += gridDim.z) {
    const double inv = inverse_norm(a.partial + (int64_t)item * kNormParts, a.parts, red);
    for (int r0 = blockIdx.y * 32; r0 < a.mp; r0 += gridDim.y * 32) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 32; k += kThreads / 32) {      // G's rows are X's columns
        const int r = c0 + ty + k, c = r0 + tx;
        tile[ty + k][tx] = r < a.rows && c < a.cols ? element(a.g, a.bf16, item * a.stride + (int64_t)r * a.cols + c) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 32; k += kThreads / 32) {
        const float x = (float)((double)tile[tx][ty + k] * inv);
        const int64_t at = ((int64_t)item * a.mp + r0 + ty + k) * a.np + c0 + tx;
        a.x[at] = x;
        reinterpret_cast<__half*>(a.xs)[at] = __float2half_rn(x * a.scale);
      }
    }
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
  const int64_t want = (n + 16383) / 16384;
  return (int)(want < 1 ? 1 : want > kNormParts ? kNormParts : want);
}
cudaError_t square_sums(const void* g, int bf16, int64_t items, int64_t n, int64_t stride, double* partial, uint32_t* clear, int zeros,
                        cudaStream_t stream) {
  const int parts = norm_parts(n);
  const int64_t per = ((n + parts - 1) / parts + 7) / 8 * 8;
  return launch_dependent(square_sums_kernel, dim3(parts, (unsigned)(items < 4096 ? items : 4096)), kSumThreads, 0, stream, g, bf16, items, n,
                          stride, per, partial, clear, zeros);
}
cudaError_t load_unit(const LoadUnit& a, cudaStream_t stream) {
  if (a.mp % 32 || a.np % 32 || a.parts > kThreads) return cudaErrorInvalidValue;
  const unsigned items = (unsigned)(a.items < 4096 ? a.items : 4096);
  // several pieces a CTA, which sums the norm's parts first
  if (a.transpose) {
    const int columns = a.np / 32, want = 148 * 16 / columns / (int)items, blocks = a.mp / 32;
    return launch_dependent(load_unit_transposed_kernel, dim3(columns, want < 1 ? 1 : want < blocks ? want : blocks, items), kThreads, 0, stream, a);
  }
  const int64_t all = ((int64_t)a.mp * (a.np / 4) + kThreads - 1) / kThreads, most = 148 * 16 / items + 1;
  return launch_dependent(load_unit_kernel, dim3((unsigned)(all < most ? all : most), items), kThreads, 0, stream, a);
}

}  // namespace msb
