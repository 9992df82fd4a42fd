// All steps of the orthogonal update of a matrix of up to 256 x 256 in one launch: a cluster of two CTAs has it in shared and tensor memory.
//
// CTA r holds rows 128 r .. 128 r + 127 of X, of A = X X^T and of b A + c A^2 as fp16 (128-byte swizzle, 64 columns a block) and X itself, times the
// products' scale, as an fp32 accumulator in tensor memory.  The three products of a step are tcgen05.mma of the pair, 256 x 256:
//   A          both factors are the rows of X as they lie;
//   A A        A is symmetric: both factors are the rows of A;
//   X' = a X + B X    the accumulator, multiplied by a, goes on; the second factor is X by columns, of which either CTA holds 128: the
//              rows are written to both CTAs.
// X is held times 32 and A times 32^2, as their products are, so that sums become factors without a multiplication: fp16 has 11 significant
// bits down to 2^-14 / 32 of X (an element of 256 x 256 is 2^-8 in the mean), and 2^-24 of what is below.
// Between the products the epilogue warps turn sums into the next factors, where the factors before lie.  Latencies bound it.  A step of 16 x 16 takes 3.5 us,
// of 64 x 64 4.9, of 256 x 256 9.7 (from calls of 1 to 20 steps, at 1.9 GHz).  Of the last the tensor pipe has 3.1, 16 instructions of 128 cycles a product;
// from one product to the next are 2200 cycles of 16 x 16 (commit and wait 500, tensor memory, conversion and shared memory 600, the fence to the tensor
// pipe's view of it 550, 1000 with stores to the other CTA, arrival and wait 300) and 4300 of 256 x 256, where a warp has 64 columns to
// convert and to store to both CTAs.  Outside the steps are 17 to 23 us: the launch and its events 6, the rest G's way from memory,
// |G| in 64 bits, the first factors, the result.  256 x 256 in five steps 66 to 71 us (101 as seventeen launches), 64 x 64 43.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../common/f32x2.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "../common/store_row.cuh"
#include "../gemm/pair.cuh"
#include "orthogonal.h"

namespace msb {

namespace {

constexpr int kSide = kUnitSide, kHalf = kSide / 2;
constexpr float kScale = 32.f;                                     // of X
constexpr int kEpiThreads = 512, kThreads = kEpiThreads + 32;      // warps 0 - 15: rows 32 (w & 3), columns 64 (w >> 2); the last issues the products
constexpr int kPart = kSide / (kEpiThreads / 128), kChunks = kPart / 32;   // columns of a warp
constexpr uint32_t kBlockRows = kHalf * 128;                       // 64 columns of a CTA's rows
constexpr uint32_t kBlockCols = kSide * 128;                       // 64 columns of all rows
constexpr uint32_t kRowBytes = kSide / 64 * kBlockRows, kColBytes = kHalf / 64 * kBlockCols;
// behind them: two barriers, both CTAs' norms, the slot of the tensor memory's address with room for another, the warps' sums
constexpr uint32_t kTail = 2 * sizeof(uint64_t) + 2 * sizeof(double) + 2 * sizeof(uint32_t) + kEpiThreads / 32 * sizeof(double);
constexpr uint32_t kSmem = 2 * kRowBytes + kColBytes + 1024 + kTail;          // the first 1024 for alignment
static_assert(kRowBytes == 65536 && kColBytes == 65536, "");

__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 floats_of(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ void store_remote(uint32_t addr, const uint4& v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// A bounded wait; what threads of either CTA did before their arrivals is seen after it (a fence of the cluster in its place takes 1000 cycles).
__device__ __forceinline__ bool arrived(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, uint64_t timeout_ns) {
  if (arrived(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 0;; ++it) {
    if (arrived(bar, parity)) return true;
    if ((it & 0x3f) == 0x3f && globaltimer_ns() - t0 > timeout_ns) return false;
  }
}
// Place of 8 columns from `col` on in row `row`, blocks of 64 columns being `block` bytes apart.
__device__ __forceinline__ uint32_t place16(int row, int col, uint32_t block) {
  return (uint32_t)(col >> 6) * block + (uint32_t)row * 128 + ((((uint32_t)col >> 3 & 7) ^ ((uint32_t)row & 7)) << 4);
}

}  // namespace

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
orthogonal_small_kernel(const UnitSmall a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* const sX = smem;                       // rows of X
  uint8_t* const sA = sX + kRowBytes;             // rows of A, then of B
  uint8_t* const sXc = sA + kRowBytes;            // this CTA's columns of X, all rows
  uint64_t* const done = reinterpret_cast<uint64_t*>(sXc + kColBytes);       // in both CTAs: the product is complete
  uint64_t* const ready = done + 1;                                // in the leader: the factors are there; an arrival of every epilogue warp
  double* const norm = reinterpret_cast<double*>(ready + 1);       // [2]: of either CTA's part
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(norm + 2);
  double* const red = reinterpret_cast<double*>(tmem_slot + 2);    // [kEpiThreads / 32]

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool epilogue = warp < kEpiThreads / 32;
  if (threadIdx.x == 0) {
    mbar_init(done, 1);
    mbar_init(ready, 2 * (kEpiThreads / 32));
    mbar_fence_init();
  }
  if (warp == kEpiThreads / 32) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_trigger();
  grid_wait();

  const int item = blockIdx.x >> 1;
  const bool tall = a.rows > a.cols;
  const int m = tall ? a.cols : a.rows, n = tall ? a.rows : a.cols;
  const int mk = (m + 15) / 16, nk = (n + 15) / 16;                // instructions of a contraction
  const int64_t base = item * a.stride;
  const auto element = [&](int64_t i) {
    return a.bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.g)[base + i]) : reinterpret_cast<const float*>(a.g)[base + i];
  };
  const int q = warp & 3, col0 = (warp >> 2) * kPart;
  const int local = q * 32 + lane, row = (int)rank * kHalf + local;
  const bool rows_here = (int)rank * kHalf + q * 32 < m;            // what lies beyond in the same 32 rows or columns is zero
  const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
  const uint32_t accA = tmem + lanes, accX = tmem + lanes + kSide;
  const uint32_t to = mapa_u32(smem_u32(sXc), rank ^ 1);

  // ---- this CTA's rows of X, not yet divided by |G|, through shared memory: read from memory along G's rows, sixteen loads a thread in flight;
  // column c of a row lies at c ^ row in its group of 32, so that rows and columns of lanes are in different banks.  |G| in 64 bits ----
  float* const staged = reinterpret_cast<float*>(sA);               // [128][256], where A and the columns of X are later
  double s = 0.0;
  if (epilogue) {
    // pass k: rows 2 k and 2 k + 1, a column a thread, or (of a tall G) columns 4 k .. 4 k + 3, a row a thread
    const int passes = tall ? (n + 3) / 4 : (min(m - (int)rank * kHalf, kHalf) + 1) / 2;
    const auto row_of = [&](int k) { return tall ? (int)threadIdx.x & (kHalf - 1) : 2 * k + ((int)threadIdx.x >> 8); };
    const auto col_of = [&](int k) { return tall ? 4 * k + ((int)threadIdx.x >> 7) : (int)threadIdx.x & (kSide - 1); };
#pragma unroll 1
    for (int k0 = 0; k0 < passes; k0 += 16) {
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int r = (int)rank * kHalf + row_of(k0 + k), j = col_of(k0 + k);
        v[k] = k0 + k < passes && r < m && j < n ? element(tall ? (int64_t)j * a.cols + r : (int64_t)r * a.cols + j) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int i = row_of(k0 + k), j = col_of(k0 + k);
        if (k0 + k < passes) staged[i * kSide + (j & ~31) + ((j ^ i) & 31)] = v[k];
        s += (double)v[k] * v[k];
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (epilogue && lane == 0) red[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int k = 0; k < kEpiThreads / 32; ++k) s += red[k];
    const uint32_t here = smem_u32(norm + rank);
    for (uint32_t r = 0; r < 2; ++r) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_u32(here, r)), "d"(s) : "memory");
  }
  float mine[kChunks][32];                                            // this thread's part of its row
  if (epilogue) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 32; ++i)
        mine[c][i] = row < m && col0 + c * 32 + i < n ? staged[local * kSide + col0 + c * 32 + ((i ^ local) & 31)] : 0.f;
  }
  cluster_sync_all();                                                 // the other CTA may write its columns there
  const double sum = norm[0] + norm[1], inverse = sum == 0.0 ? 0.0 : 1.0 / sqrt(sum);

  // 32 columns of X from `col` on: its fp16 copies, and the accumulator of the next step
  const auto write_x = [&](const float (&v)[32], int col) {
    const bool own = col0 / kHalf == (int)rank;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 w = make_uint4(half2_of(v[8 * k], v[8 * k + 1]), half2_of(v[8 * k + 2], v[8 * k + 3]), half2_of(v[8 * k + 4], v[8 * k + 5]),
                                 half2_of(v[8 * k + 6], v[8 * k + 7]));
      *reinterpret_cast<uint4*>(sX + place16(local, col + 8 * k, kBlockRows)) = w;
      const uint32_t at = place16(row, (col & (kHalf - 1)) + 8 * k, kBlockCols);
      if (own) *reinterpret_cast<uint4*>(sXc + at) = w;
      else store_remote(to + at, w);
    }
    uint32_t r[32];
    const uint64_t f = f32x2(a.a, a.a);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float lo, hi;
      split(mul2(f32x2(v[2 * i], v[2 * i + 1]), f), lo, hi);
      r[2 * i] = __float_as_uint(lo);
      r[2 * i + 1] = __float_as_uint(hi);
    }
    __syncwarp();
    tmem_st_32x32(accX + col, r);
  };
  const auto read = [&](uint32_t from, float (&v)[32]) {
    uint32_t r[32];
    __syncwarp();
    tmem_ld_32x32(from, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  };
  const uint32_t ready_leader = mapa_u32(smem_u32(ready), 0);
  // What this warp wrote, here and in the other CTA, is there for the next product; what it read may be overwritten.
  const auto handed_over = [&](bool remote) {
    if (remote) asm volatile("fence.proxy.async.shared::cluster;" ::: "memory");
    else fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(ready_leader) : "memory");
  };

  if (epilogue) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = col0 + c * 32;
#pragma unroll
      for (int i = 0; i < 32; ++i) mine[c][i] = (float)((double)mine[c][i] * inverse) * kScale;
      if (rows_here && col < n) write_x(mine[c], col);
    }
    tmem_st_wait();
    handed_over(true);
  }

  const uint64_t rows_x = make_smem_desc(smem_u32(sX), 16, 1024), rows_a = make_smem_desc(smem_u32(sA), 16, 1024);
  const uint64_t cols_x = make_smem_desc(smem_u32(sXc), kBlockCols, 1024);
  constexpr uint32_t kFormats = (1u << 7) | (1u << 10);                            // bf16 of both factors, taken out: fp16
  const uint32_t plain = make_idesc_bf16(kSide, kSide, 0, 0) & ~kFormats, by_columns = make_idesc_bf16(kSide, kSide, 0, 1) & ~kFormats;
  bool ok = true;
  uint32_t phase = 0;
  // Bounded.  A thread that has given up does no more work and still comes to the end.
  const auto finished = [&](uint64_t* bar) {
    if (ok && !wait_cluster(bar, phase, a.timeout_ns)) {
      ok = false;
      if (atomicCAS(a.status, 0u, kUnitTimeout) == 0u) {
        a.status[1] = blockIdx.x;
        a.status[2] = (uint32_t)warp;
        a.status[3] = phase;
      }
    }
    phase ^= 1;
    return ok;
  };
  // The same for a warp: one lane waits.  A shuffle orders no memory; what orders the other lanes behind the wait is the warp barrier that every
  // read of tensor memory begins with (one here as well: 1.4 us of 67).
  const auto complete = [&]() {
    int there = 1;
    if (lane == 0) there = finished(done) ? 1 : 0;
    there = __shfl_sync(0xffffffffu, there, 0);
    tc_fence_after_sync();
    return there != 0;
  };
  // K-major: 16 elements are 32 bytes of a block's rows; four of them, then the next block.  By columns: 16 rows of 128 bytes.
  const auto product = [&](uint32_t acc, uint64_t fa, uint64_t fb, bool columns, int k16, bool go_on) {
    if (!finished(ready)) return;
    tc_fence_after_sync();
    for (int k = 0; k < k16; ++k) {
      const uint32_t step = (uint32_t)(k >> 2) * (kBlockRows >> 4) + (uint32_t)(k & 3) * 2;
      umma_f16_pair(acc, fa + step, fb + (columns ? (uint32_t)k * (16 * 128 >> 4) : step), columns ? by_columns : plain, go_on || k > 0 ? 1u : 0u);
    }
    umma_commit_both(smem_u32(done));
  };
  if (!epilogue) {
    if (rank == 0 && elect_one())
      for (int step = 0; step < a.steps; ++step) {
        product(tmem, rows_x, rows_x, false, nk, false);
        product(tmem, rows_a, rows_a, false, mk, false);
        product(tmem + kSide, rows_a, cols_x, true, mk, true);
      }
  } else {
#pragma unroll 1
    for (int step = 0; step < a.steps; ++step) {
      const bool last = step + 1 == a.steps;
      if (complete()) {
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          const int col = col0 + c * 32;
          if (!rows_here || col >= m) break;
          float v[32];
          read(accA + col, v);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(sA + place16(local, col + 8 * k, kBlockRows)) =
                make_uint4(half2_of(v[8 * k], v[8 * k + 1]), half2_of(v[8 * k + 2], v[8 * k + 3]), half2_of(v[8 * k + 4], v[8 * k + 5]),
                           half2_of(v[8 * k + 6], v[8 * k + 7]));
        }
      }
      handed_over(false);
      if (complete()) {
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          const int col = col0 + c * 32;
          if (!rows_here || col >= m) break;
          float v[32];
          read(accA + col, v);
          // A lies times 32^2, the sums are times 32^4
          constexpr float kA = 1.f / (kScale * kScale);
          const uint64_t f = f32x2(a.c * kA * kA, a.c * kA * kA), h = f32x2(a.b * kA, a.b * kA);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint4* const at = reinterpret_cast<uint4*>(sA + place16(local, col + 8 * k, kBlockRows));
            const uint4 x = *at;
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 t = floats_of(w[i]);
              float lo, hi;
              split(fma2(h, f32x2(t.x, t.y), mul2(f, f32x2(v[8 * k + 2 * i], v[8 * k + 2 * i + 1]))), lo, hi);
              o[i] = half2_of(lo, hi);
            }
            *at = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
      handed_over(false);
      if (complete()) {
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          const int col = col0 + c * 32;
          if (!rows_here || col >= n) break;
          float v[32];
          read(accX + col, v);
          if (!last) {
            write_x(v, col);
          } else if (row < m) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= 1.f / kScale;
            store_row32(a.out, item * a.out_item + row * (tall ? a.out_col : a.out_row) + col * (tall ? a.out_row : a.out_col),
                        tall ? a.out_row : a.out_col, min(32, n - col), a.out_fp32 != 0, v);
          }
        }
        if (!last) tmem_st_wait();
      }
      if (!last) handed_over(true);
    }
  }
  // both CTAs are done with shared and tensor memory of the pair
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  if (warp == kEpiThreads / 32) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

cudaError_t orthogonal_small(const UnitSmall& a, cudaStream_t stream) {
  if (a.rows < 1 || a.cols < 1 || a.rows > kSide || a.cols > kSide || a.items < 1 || a.items > (1 << 29)) return cudaErrorInvalidValue;
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(orthogonal_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  return launch_dependent(orthogonal_small_kernel, 2 * a.items, kThreads, kSmem, stream, a);
}

}  // namespace msb
