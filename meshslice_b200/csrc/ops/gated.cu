#include <cuda_bf16.h>

#include "../common/gate.cuh"
#include "../common/pdl.cuh"
#include "gated.h"

namespace msb {

namespace {

__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kThreads = 256;

}  // namespace

// HBM bounds both: 6 and 10 bytes an element, a thread takes 16 bytes of each operand.
__global__ void __launch_bounds__(kThreads)
gated_act_kernel(const uint4* g, const uint4* u, uint4* h, int64_t nvec, int act) {
  grid_trigger();
  grid_wait();
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < nvec; i += (int64_t)gridDim.x * kThreads) {
    float a[8], b[8];
    unpack(g[i], a);
    unpack(u[i], b);
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = a[k] * gate_sigmoid(a[k], act) * b[k];
    h[i] = pack(a);
  }
}
__global__ void __launch_bounds__(kThreads)
gated_act_bwd_kernel(const uint4* dh, const uint4* g, const uint4* u, uint4* dg, uint4* du, int64_t nvec, int act) {
  grid_trigger();
  grid_wait();
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < nvec; i += (int64_t)gridDim.x * kThreads) {
    float a[8], b[8], d[8], e[8];
    unpack(dh[i], d);
    unpack(g[i], a);
    unpack(u[i], b);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float s = gate_sigmoid(a[k], act);
      e[k] = d[k] * (a[k] * s);             // the bounded factor first: without it the others may leave fp32 where it is 0
      d[k] = d[k] * (b[k] * gate_slope(a[k], s, act));
    }
    dg[i] = pack(d);
    du[i] = pack(e);
  }
}

static int grid_of(int64_t nvec) {
  const int64_t want = (nvec + kThreads - 1) / kThreads;
  return (int)(want < (1 << 22) ? want : 1 << 22);
}
cudaError_t gated_act(const void* g, const void* u, void* h, int64_t n, int act, cudaStream_t stream) {
  if (n % 8) return cudaErrorInvalidValue;
  return launch_dependent(gated_act_kernel, grid_of(n / 8), kThreads, 0, stream, reinterpret_cast<const uint4*>(g),
                          reinterpret_cast<const uint4*>(u), reinterpret_cast<uint4*>(h), n / 8, act);
}
cudaError_t gated_act_bwd(const void* dh, const void* g, const void* u, void* dg, void* du, int64_t n, int act, cudaStream_t stream) {
  if (n % 8) return cudaErrorInvalidValue;
  return launch_dependent(gated_act_bwd_kernel, grid_of(n / 8), kThreads, 0, stream, reinterpret_cast<const uint4*>(dh),
                          reinterpret_cast<const uint4*>(g), reinterpret_cast<const uint4*>(u), reinterpret_cast<uint4*>(dg),
                          reinterpret_cast<uint4*>(du), n / 8, act);
}

}  // namespace msb
