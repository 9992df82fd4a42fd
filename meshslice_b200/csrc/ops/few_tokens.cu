// The weights bound these products: 2 bytes an element for 2 T operations, which a tile of the tcgen05 pipe would spend on 256 rows, T of them
// tokens.  Here the weights go from memory into the registers of mma.sync (rows: outputs, columns: 8 tokens), 16 bytes a load and in the
// order in which they lie: what the instruction takes for consecutive positions of the contraction, or for neighbouring outputs, may be any,
// as long as both operands agree and the results are put where they belong.  The warps of a CTA and the CTAs of a cluster take parts of the
// contraction; their sums meet in shared memory.  With fp32 arithmetic on the same loads 8 tokens took 24 us at 1024 x 2816.
#include <cuda_bf16.h>

#include "../common/gate.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "few_tokens.h"

namespace msb {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;

// D += A B of 16 x 16 and 16 x 8.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A unit of the contraction that ends within it is loaded without a question, which would be a branch, for each load, and all of it is in flight.  A plain
// product of 28672 x 8192 and one token takes 125 instead of 193 us, of 16 tokens and weights [N, K] 110 instead of 156; of a gated one, whose
// CTAs are many, the same loads took 197 instead of 179 (4096 x 10752 37.6 instead of 35.3): it keeps the questions.
template <bool kWhole>
struct Whole {
  static constexpr bool value = kWhole;
};
__device__ __forceinline__ uint4 load_if(bool there, const void* p) {
  return there ? ld_stream(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ uint32_t ctas() {
  uint32_t v;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(v));
  return v;
}
__device__ __forceinline__ float shared_of(const float* p, uint32_t rank) {
  uint32_t a = smem_u32(p), b;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(b) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The sums of the warps [kWarps][rows][8 G] of every CTA of the cluster, joined in the order of the contraction's parts.  Columns [0, half) are
// the gate's of as many outputs, the others the up projection's (a plain product: all are outputs); row(c) is where column c lies.
template <int G, bool kGated, int kRows, class Row>
__device__ __forceinline__ void join(const FewTokens& a, float* sums, int block, Row row) {
  constexpr int kT = 8 * G, kOuts = kGated ? kRows / 2 : kRows;
  const uint32_t size = ctas(), rank = blockIdx.x % size;
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kT; i += kThreads) {
    float s = sums[i];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s += sums[w * kRows * kT + i];
    sums[i] = s;
  }
  if (size > 1) cluster_barrier();
  else __syncthreads();
  for (int i = threadIdx.x + rank * kThreads; i < kOuts * kT; i += kThreads * size) {
    const int t = i / kOuts, c = i % kOuts, out = block * kOuts + c;
    if (t >= a.tokens || out >= a.N) continue;
    float g = 0.f, u = 0.f;
    for (uint32_t r = 0; r < size; ++r) {
      g += shared_of(sums + row(c) * kT + t, r);
      if (kGated) u += shared_of(sums + row(c + kOuts) * kT + t, r);
    }
    if (kGated) g = g * gate_sigmoid(g, a.act) * u;
    reinterpret_cast<__nv_bfloat16*>(a.out)[t * a.ldo + out] = __float2bfloat16_rn(g);
  }
  if (size > 1) cluster_barrier();      // the others may still read this CTA's sums
}

}  // namespace

// Weights [N, K]: 16 rows a CTA (of a gated product 8 of either matrix).  A lane has rows g and g + 8 and token g, and 8 elements of each at
// 8 tg of every 32: two instructions' worth.
constexpr int kNtRows = 16, kNtUnit = 128;
template <int G, bool kGated>
__global__ void __launch_bounds__(kThreads)
few_nt_kernel(const FewTokens a) {
  grid_trigger();
  grid_wait();
  __shared__ float sums[kWarps * kNtRows * 8 * G];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tg = lane & 3;
  const int size = (int)ctas(), part = (int)(blockIdx.x % size) * kWarps + warp, block = blockIdx.x / size;
  const int first = block * (kGated ? 8 : 16);
  const __nv_bfloat16* const w0 = reinterpret_cast<const __nv_bfloat16*>(a.w) + (int64_t)min(first + g, a.N - 1) * a.ldw;   // rows beyond the last are not stored
  const __nv_bfloat16* const w1 = kGated ? reinterpret_cast<const __nv_bfloat16*>(a.up) + (int64_t)min(first + g, a.N - 1) * a.ldu
                                         : reinterpret_cast<const __nv_bfloat16*>(a.w) + (int64_t)min(first + 8 + g, a.N - 1) * a.ldw;
  const __nv_bfloat16* x[G];
#pragma unroll
  for (int i = 0; i < G; ++i) x[i] = reinterpret_cast<const __nv_bfloat16*>(a.x) + (int64_t)min(8 * i + g, a.tokens - 1) * a.ldx;
  float d[G][4] = {};
  const auto unit = [&](int k0, auto whole) {
    const auto there = [&](int k) { return decltype(whole)::value || k < a.K; };
    uint4 p[4], q[4], v[G][4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int k = k0 + 32 * f + 8 * tg;
      p[f] = load_if(there(k), w0 + k);
      q[f] = load_if(there(k), w1 + k);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int k = k0 + 32 * f + 8 * tg;
#pragma unroll
      for (int i = 0; i < G; ++i) v[i][f] = there(k) ? *reinterpret_cast<const uint4*>(x[i] + k) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int i = 0; i < G; ++i) {
        mma(d[i], p[f].x, q[f].x, p[f].y, q[f].y, v[i][f].x, v[i][f].y);
        mma(d[i], p[f].z, q[f].z, p[f].w, q[f].w, v[i][f].z, v[i][f].w);
      }
  };
  int k0 = part * kNtUnit;
  if (!kGated)
    for (; k0 + kNtUnit <= a.K; k0 += size * kWarps * kNtUnit) unit(k0, Whole<true>{});
  for (; k0 < a.K; k0 += size * kWarps * kNtUnit) unit(k0, Whole<false>{});
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[(warp * kNtRows + g + 8 * (j >> 1)) * 8 * G + 8 * i + 2 * tg + (j & 1)] = d[i][j];
  join<G, kGated, kNtRows>(a, sums, block, [](int c) { return c; });
}

// Weights [K, N]: 64 columns a CTA (of a gated product 32 of either matrix).  A lane has columns 8 g .. 8 g + 7, in rows 4 tg .. 4 tg + 3 of
// every 16, whose neighbours it packs into pairs: instruction j takes columns 8 g + j and 8 g + j + 4.
constexpr int kNnRows = 64, kNnUnit = 32;
template <int G, bool kGated>
__global__ void __launch_bounds__(kThreads)
few_nn_kernel(const FewTokens a) {
  grid_trigger();
  grid_wait();
  __shared__ float sums[kWarps * kNnRows * 8 * G];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tg = lane & 3;
  const int size = (int)ctas(), part = (int)(blockIdx.x % size) * kWarps + warp, block = blockIdx.x / size;
  const bool second = kGated && g >= 4;
  const int col = kGated ? block * 32 + 8 * (g & 3) : block * 64 + 8 * g;
  const int64_t ld = second ? a.ldu : a.ldw;
  const __nv_bfloat16* const w = reinterpret_cast<const __nv_bfloat16*>(second ? a.up : a.w) + min(col, a.N - 8);   // columns beyond the last are not stored
  const __nv_bfloat16* x[G];
#pragma unroll
  for (int i = 0; i < G; ++i) x[i] = reinterpret_cast<const __nv_bfloat16*>(a.x) + (int64_t)min(8 * i + g, a.tokens - 1) * a.ldx;
  float d[G][4][4] = {};
  const auto unit = [&](int k0, auto whole) {
    const auto there = [&](int k) { return decltype(whole)::value || k < a.K; };
    uint4 p[2][4];
    uint2 v[G][2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int k = k0 + 16 * f + 4 * tg;              // K is a multiple of 8: four rows there or none
#pragma unroll
      for (int r = 0; r < 4; ++r) p[f][r] = load_if(there(k), w + (k + r) * ld);
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int k = k0 + 16 * f + 4 * tg;
#pragma unroll
      for (int i = 0; i < G; ++i) v[i][f] = there(k) ? *reinterpret_cast<const uint2*>(x[i] + k) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto near = [&](const uint4& u) { return j < 2 ? u.x : u.y; };
        const auto far = [&](const uint4& u) { return j < 2 ? u.z : u.w; };
        const uint32_t pick = j & 1 ? 0x7632 : 0x5410;       // the upper or the lower halves of two rows
        const uint32_t a0 = __byte_perm(near(p[f][0]), near(p[f][1]), pick), a1 = __byte_perm(far(p[f][0]), far(p[f][1]), pick);
        const uint32_t a2 = __byte_perm(near(p[f][2]), near(p[f][3]), pick), a3 = __byte_perm(far(p[f][2]), far(p[f][3]), pick);
#pragma unroll
        for (int i = 0; i < G; ++i) mma(d[i][j], a0, a1, a2, a3, v[i][f].x, v[i][f].y);
      }
  };
  int k0 = part * kNnUnit;
  if (!kGated)
    for (; k0 + kNnUnit <= a.K; k0 += size * kWarps * kNnUnit) unit(k0, Whole<true>{});
  for (; k0 < a.K; k0 += size * kWarps * kNnUnit) unit(k0, Whole<false>{});
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) sums[(warp * kNnRows + 8 * (j + 4 * (c >> 1)) + g) * 8 * G + 8 * i + 2 * tg + (c & 1)] = d[i][j][c];
  // row 8 j + g holds column 8 g + j: neighbouring lanes write neighbouring words
  join<G, kGated, kNnRows>(a, sums, block, [](int c) { return (c & 7) << 3 | c >> 3; });
}

// CTAs of a cluster.  It costs some 2 us beside a plain launch: 8 tokens of 1024 x 2816, weights [K, N], 16.3, 15.8 and 17.4 us with at least 32, 64 and
// 148 CTAs.  Where every warp keeps two units of the contraction, two CTAs an SM are worth more (one with 9 tokens or more, whose CTAs take twice the
// registers): one token of 10752 x 4096, down weight [K, N], 95 us with 64 CTAs and 62 with 512, of 28672 x 8192 314 with 128 and 139 with 512.
static int cluster_of(int64_t blocks, int64_t units, int64_t most) {
  int size = 1;
  while (size < 8 && ((blocks * size < 64 && 2 * size * kWarps <= units) || (blocks * size < most && 4 * size * kWarps <= units))) size *= 2;
  return size;
}

template <int G, bool kGated>
static cudaError_t launch_few(const FewTokens& a, cudaStream_t stream) {
  const int64_t most = G == 1 ? 296 : 148;
  if (a.nt) {
    const int outs = kGated ? 8 : 16, blocks = (a.N + outs - 1) / outs, size = cluster_of(blocks, (a.K + kNtUnit - 1) / kNtUnit, most);
    const auto kernel = few_nt_kernel<G, kGated>;
    return launch_dependent_clusters(kernel, size, dim3(blocks * size), kThreads, 0, stream, a);
  }
  const int outs = kGated ? 32 : 64, blocks = (a.N + outs - 1) / outs, size = cluster_of(blocks, (a.K + kNnUnit - 1) / kNnUnit, most);
  const auto kernel = few_nn_kernel<G, kGated>;
  return launch_dependent_clusters(kernel, size, dim3(blocks * size), kThreads, 0, stream, a);
}

cudaError_t few_tokens(const FewTokens& a, cudaStream_t stream) {
  if (a.tokens < 1 || a.tokens > kFewTokens || a.K % 8 || a.N % 8) return cudaErrorInvalidValue;
  if (a.up != nullptr) return a.tokens <= 8 ? launch_few<1, true>(a, stream) : launch_few<2, true>(a, stream);
  return a.tokens <= 8 ? launch_few<1, false>(a, stream) : launch_few<2, false>(a, stream);
}

}  // namespace msb
