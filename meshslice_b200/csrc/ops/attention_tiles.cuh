// What the attention kernels share: 128 x 128 bf16 tiles in swizzled shared memory and tensor memory, exponentials, cluster
// launch control.
#pragma once
#include <cuda_bf16.h>

#include "../common/ptx.cuh"

namespace msb {

namespace {

constexpr int kD = 128;         // head dim
constexpr int kBlk = 128;       // query / key rows per tile
constexpr int kTile = kBlk * kD * 2;  // 32 KiB: one [128 x 128] bf16 tile = two swizzle halves
constexpr int kHalf = kTile / 2;
// A warp may touch the TMEM lanes 32 * (warp % 4) ... + 31: any four consecutive warps cover the 128 rows of a tile, whichever
// warp the element-wise work starts at.
constexpr uint32_t kErrAttn = 20;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void report(uint32_t* status, uint32_t code, uint32_t d0, uint32_t d1) {
  if (atomicCAS(status, 0u, code) == 0u) {
    status[1] = blockIdx.x + (blockIdx.y << 12) + (blockIdx.z << 22);
    status[2] = d0;
    status[3] = d1;
  }
}

// Bounded wait of a whole warp: the lanes poll together (one transaction), the verdict is common.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint64_t tmo) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, tmo));
}

// 2^x on the special-function unit in one instruction (relative error 2^-22, denormal results
// flushed to zero: probabilities below 2^-126 are zero anyway).  exp2f() wraps the same
// instruction in range scaling that costs several more issue slots per element.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// K-major view of a tile: rows = M or N index, contraction along the 128 columns.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t tile, int kstep) {
  return make_smem_desc(tile + (kstep >> 2) * kHalf + (kstep & 3) * 32, 16, 1024);
}
// MN-major view: rows = contraction index (16 per step), the 128 columns are the M or N index.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t tile, int kstep) {
  return make_smem_desc(tile + kstep * 2048, kHalf, 1024);
}

// Cluster launch control: ask for a block of this grid that has not been launched (16-byte response into shared
// memory, announced on an mbarrier); after a refusal nothing more may be asked.
__device__ __forceinline__ void clc_try_cancel(void* resp, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(resp)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool clc_read(const void* resp, uint32_t& x, uint32_t& y, uint32_t& z) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %3, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, %2, _}, r;\n\t}"
      : "=&r"(x), "=&r"(y), "=&r"(z), "=&r"(ok) : "r"(smem_u32(resp)) : "memory");
  return ok != 0;
}

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns: thread t of the warp writes row (lane base + t).
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 16 lanes x 32 fp32 columns in the layout of a matrix fragment: thread t gets, of every group n of 8 columns, columns
// 2 (t % 4) and + 1 of rows t / 4 (r[4n], r[4n + 1]) and t / 4 + 8 (r[4n + 2], r[4n + 3]).
__device__ __forceinline__ void tmem_ld_16x32_frag(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// The same elements as packed bf16: r[2n] / r[2n + 1] are the two columns of rows t / 4 / t / 4 + 8; groups of 8 columns: 4 or 2.
__device__ __forceinline__ void tmem_st_16x32_frag(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_16x16_frag(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// The staging area may be written again: the copy engine has read it.
__device__ __forceinline__ void warp_stage_free() {
  if ((threadIdx.x & 31) == 0) bulk_wait_read<0>();
  __syncwarp();
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace

}  // namespace msb
