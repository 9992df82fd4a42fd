// Window attention with first tokens that stay visible, forward and backward, on tcgen05: the kernels of attention.cu over lists of
// key blocks instead of prefixes, for shared key/value heads and sequences that end inside a tile.
//
// A query block's list holds the blocks of the first tokens and those of its window; blocks between them are never loaded.  A key block
// is streamed by the query blocks of its window, or by all later ones where it holds a first token, of every query head of its group:
// shared heads add up in tensor memory.  Tensor maps end with their sequence (three dimensions), so rows beyond it are zeros when
// read, and left alone when written.
// All waits are bounded; a timeout records a code in `status` and the CTA leaves.
#include "window_attention.h"

#include <cuda_bf16.h>

#include "../common/f32x2.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "../gemm/sm100_gemm.h"  // make_tensor_map_seq
#include "attention_tiles.cuh"

namespace msb {

namespace {

constexpr uint32_t kErrWindow = 40;
constexpr int kThinKeys = 16;       // few first tokens: the narrowest product with 128 rows

struct WinArgs {
  int batch, seq, kv, group, heads;   // heads = kv * group
  int window, sinks;                  // 1 <= window <= seq, 0 <= sinks <= seq
  float scale;
  float* lse;
  int tiles_per_item;                 // query tiles that a CTA works on at a time (1 or 2)
  int thin;                           // no more than kThinKeys first tokens
  uint32_t* status;
  uint64_t timeout_ns;
};

// First columns of a query head and of a key head (values follow).
template <class A>
__device__ __forceinline__ int col_q(const A& a, int h) {
  const int kv = h / a.group;
  return (kv * (a.group + 2) + h - kv * a.group) * kD;
}
template <class A>
__device__ __forceinline__ int col_q(const A& a, int kv, int h) { return (kv * (a.group + 2) + h - kv * a.group) * kD; }
template <class A>
__device__ __forceinline__ int col_k(const A& a, int kv) { return (kv * (a.group + 2) + a.group) * kD; }
// First key block of query block i's window, blocks that hold first tokens.
template <class A>
__device__ __forceinline__ int window_block(const A& a, int i) { return max(0, i * kBlk - a.window + 1) / kBlk; }
template <class A>
__device__ __forceinline__ int sink_blocks(const A& a) { return (a.sinks + kBlk - 1) / kBlk; }

// 32 lanes x 16 / 8 consecutive 32-bit columns: thread t of the warp has row (lane base + t).
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// n low bits, for any n.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// 2^x of two lanes on the FMA pipe, for the share of the exponentials that would queue for the special-function unit: x = n + f with n
// the nearest whole number, 2^f by the polynomial of degree 5 with the smallest largest relative error on [-1/2, 1/2] (Remez exchange;
// 2^-23.7, with fp32 rounding 2^-22.2), times 2^n.  (n added to the exponent's bits would make a NaN the largest number.)  Below -125
// the result is about 2^-125 and not zero; NaN stays NaN.  x stays below 127 wherever the result is used.
__device__ __forceinline__ void exp2_poly(uint64_t x, float& a, float& b) {
  split(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-125.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-125.0f));
  const uint64_t t = f32x2(a, b), big = f32x2(12582912.0f, 12582912.0f);   // 1.5 * 2^23: n in the low bits
  const uint64_t r = add2(t, big), n = add2(r, f32x2(-12582912.0f, -12582912.0f)), f = fma2(n, f32x2(-1.f, -1.f), t);
  uint64_t p = f32x2(1.327647245e-03f, 1.327647245e-03f);
  p = fma2(p, f, f32x2(9.675540961e-03f, 9.675540961e-03f));
  p = fma2(p, f, f32x2(5.550713092e-02f, 5.550713092e-02f));
  p = fma2(p, f, f32x2(2.402212024e-01f, 2.402212024e-01f));
  p = fma2(p, f, f32x2(6.931469440e-01f, 6.931469440e-01f));
  p = fma2(p, f, f32x2(1.000000119e+00f, 1.000000119e+00f));
  split(r, a, b);
  split(mul2(p, f32x2(__int_as_float((__float_as_int(a) << 23) + 0x3f800000), __int_as_float((__float_as_int(b) << 23) + 0x3f800000))), a, b);
}

__device__ __forceinline__ void load_half(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int col, int row, int b) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(col), "r"(row), "r"(b)
      : "memory");
}
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int col, int row, int b) {
  load_half(dst, map, bar, col, row, b);
  load_half(dst + kHalf, map, bar, col + 64, row, b);
}
// A warp's staged box on its way, if it begins inside the sequence: every lane's writes are visible to the copy engine before lane
// 0 starts it.
__device__ __forceinline__ void warp_store_box(const CUtensorMap* map, const void* stage, int col, int row, int b, int seq) {
  fence_proxy_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0 && row < seq) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(smem_u32(stage)), "r"(col), "r"(row), "r"(b) : "memory");
    bulk_commit();
  }
}

// ==========================================================================================
// forward
// ==========================================================================================
// softmax(q k^T scale) v with the running maximum and sum of each row, in the log2 domain: m and l rescaled when the maximum grows by more
// than 2^8, one division at the end.  P is rounded to bf16 as the operand of P V (its sum l is not), the output once.
// Roles and tensor memory as in attn_fwd2_kernel: producer, MMA issuer, a softmax warpgroup for each of two neighbouring query
// tiles.  Both tiles walk one list of key blocks through the same K / V rings; each leaves out what it does not see.
// What bounds it: a step of both tiles takes 3260 cycles (2048 of the special-function unit, 1024 of products a tile), a masked block 650
// more, an item's end 2900 in which the output leaves and nothing is multiplied; below windows of about 200, HBM.  4 x 2048, 32 heads: window
// 128 54 us (6.2 TB/s), 512 with 4 first tokens 90; 1 x 16384, 16 heads on 4, window 4096 405 us (1190 TFLOP/s; under the power cap 468).
// The 90 us were 102 with first tokens as whole blocks, 97 with tile 1's own block at the head of the list.
constexpr int kFwdWarpStage = 32 * 128;   // output staging per softmax warp: 32 rows x 64 columns
constexpr size_t kFwdSmem = 6 * kTile + 8 * kFwdWarpStage + 256 + 1024;
constexpr int kFwdThreads = 384;
// registers per thread: 384 threads launch with 168; warps 0-3 give up what the softmax warps take
constexpr int kFwdRegsLow = 96, kFwdRegsHigh = 200;
static_assert(kFwdRegsLow + 2 * kFwdRegsHigh <= 3 * 168, "register shares exceed what the CTA is launched with");

// One or two neighbouring tiles (tile 0 the later one, block hi) of a head, and the list of key blocks that either sees: `ns` blocks
// with first tokens, what both have of the window from `lo` on, block hi, which tile 1 does not see, and (extra) the block before `lo`,
// which tile 0 does not see, so that each tile has one of the last two while the other has the other.  thin bit t: entry 0 holds nothing
// but first tokens, at most kThinKeys, for tile t, which takes its first kThinKeys keys only.
struct FwdItem {
  int b, h, hi, two, ns, lo, n, extra, thin;
  __device__ __forceinline__ int block(int x) const { return x < ns ? x : x + extra == n ? lo - 1 : lo + x - ns; }
  __device__ __forceinline__ bool uses(int t, int x) const { return t == 0 ? x + extra < n : two && x + 1 + extra != n; }
  __device__ __forceinline__ int first(int t) const { return t == 1 && n == 2 && extra ? 1 : 0; }
  __device__ __forceinline__ int last(int t) const { return t == 0 ? n - 1 - extra : extra ? n - 1 : n - 2; }
  __device__ __forceinline__ int next(int t, int x) const { return t == 1 && x + 2 + extra == n ? x + 2 : x + 1; }
};
__device__ __forceinline__ FwdItem fwd_item(const WinArgs& a, uint32_t x, uint32_t y, uint32_t z, int group) {
  FwdItem w;
  const int bh = (int)z * group + (int)x, nblk = (a.seq + kBlk - 1) / kBlk;
  w.b = bh / a.heads;
  w.h = bh - w.b * a.heads;
  w.hi = nblk - 1 - (int)y * a.tiles_per_item;
  w.two = a.tiles_per_item == 2 && w.hi > 0 ? 1 : 0;
  w.ns = min(sink_blocks(a), w.hi + 1);
  const int lo0 = window_block(a, w.hi), lo1 = window_block(a, max(w.hi - 1, 0));
  w.lo = max(w.ns, lo0);
  w.extra = w.two && max(w.ns, lo1) < w.lo ? 1 : 0;
  w.n = w.ns + max(0, w.hi + 1 - w.lo) + w.extra;
  w.thin = a.thin && w.ns == 1 ? (lo0 > 0 ? 1 : 0) | (w.two && lo1 > 0 ? 2 : 0) : 0;
  return w;
}

__global__ void __launch_bounds__(kFwdThreads, 1)
window_fwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_out,
                  const __grid_constant__ CUtensorMap tm_thin, const __grid_constant__ WinArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                 // [2] tiles
  uint8_t* sK = smem + 2 * kTile;     // [2] stages
  uint8_t* sV = smem + 4 * kTile;     // [2] stages
  uint8_t* sO = smem + 6 * kTile;     // [8] warps
  uint64_t* bars = reinterpret_cast<uint64_t*>(sO + 8 * kFwdWarpStage);
  uint8_t* clc_resp = reinterpret_cast<uint8_t*>(bars);   // 16 bytes
  uint64_t* clc_full = bars + 2;
  uint64_t* clc_empty = bars + 3;
  uint64_t* q_full = bars + 4;        // all [2] from here
  uint64_t* q_empty = bars + 6;
  uint64_t* k_full = bars + 8;
  uint64_t* k_empty = bars + 10;
  uint64_t* v_full = bars + 12;
  uint64_t* v_empty = bars + 14;
  uint64_t* s_full = bars + 16;
  uint64_t* o_done = bars + 18;
  uint64_t* p_ready = bars + 20;      // [2 * tile + part]: columns [0,96) / [96,128) of P
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  uint64_t* item_full = bars + 25;    // the next item, as the producer has worked it out
  int4* item_slot = reinterpret_cast<int4*>(bars + 26);   // [3]

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint64_t tmo = a.timeout_ns;
  const int group = gridDim.x;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_qkv);
    mbar_init(clc_full, 1);
    mbar_init(item_full, 1);
    mbar_init(clc_empty, 9);          // MMA thread, 8 softmax warps
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(o_done + i, 1);
      mbar_init(p_ready + 2 * i, 128);
      mbar_init(p_ready + 2 * i + 1, 128);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_trigger();
  grid_wait();

  // The next item, which the producer has worked out for all: false when there is none (or on a timeout).
  uint32_t items = 0;
  auto next_item = [&](FwdItem& w) -> bool {
    if (!mbar_wait(item_full, items & 1, 8 * tmo)) {
      report(a.status, kErrWindow + 6, 0, 0);
      return false;
    }
    ++items;
    const int4 i0 = item_slot[0], i1 = item_slot[1], i2 = item_slot[2];
    w.b = i0.x; w.h = i0.y; w.hi = i0.z; w.two = i0.w;
    w.ns = i1.x; w.lo = i1.y; w.n = i1.z; w.extra = i1.w;
    w.thin = i2.x;
    return i2.y != 0;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFwdRegsLow));
    FwdItem w = fwd_item(a, blockIdx.x, blockIdx.y, blockIdx.z, group);
    if (warp == 0 && elect_one()) {
      uint32_t c = 0;                 // K / V tiles loaded so far
      uint32_t qc[2] = {0, 0};        // Q tiles loaded so far
      bool ok = true, more = true;
      while (ok && more) {
        const int colq = col_q(a, w.h), colk = col_k(a, w.h / a.group);
        for (int t = 0; t < 1 + w.two && ok; ++t) {
          if (!(ok = mbar_wait(q_empty + t, (qc[t] & 1) ^ 1, 8 * tmo))) break;
          ++qc[t];
          mbar_expect_tx(q_full + t, kTile);
          load_tile(sQ + t * kTile, &tm_qkv, q_full + t, colq, (w.hi - t) * kBlk, w.b);
        }
        for (int x = 0; x < w.n && ok; ++x, ++c) {
          const uint32_t st = c & 1, ph = ((c >> 1) & 1) ^ 1;
          const int krow = w.block(x) * kBlk;
          const bool thin = x == 0 && w.thin == (w.two ? 3 : 1);        // for all that use it
          const CUtensorMap* map = thin ? &tm_thin : &tm_qkv;
          const uint32_t bytes = thin ? kThinKeys * kD * 2 : kTile;
          if (!(ok = mbar_wait(k_empty + st, ph, 8 * tmo))) break;
          mbar_expect_tx(k_full + st, bytes);
          load_tile(sK + st * kTile, map, k_full + st, colk, krow, w.b);
          if (!(ok = mbar_wait(v_empty + st, ph, 8 * tmo))) break;
          mbar_expect_tx(v_full + st, bytes);
          load_tile(sV + st * kTile, map, v_full + st, colk + kD, krow, w.b);
        }
        // Only now, with the item's last loads on their way, ask for the next item: a CTA that took one item ahead
        // would hold it back from a CTA that is free sooner.
        if (ok && (ok = mbar_wait(clc_empty, (items & 1) ^ 1, 8 * tmo))) {
          mbar_expect_tx(clc_full, 16);
          clc_try_cancel(clc_resp, clc_full);
          uint32_t x, y, z;
          if ((ok = mbar_wait(clc_full, items & 1, 8 * tmo))) {
            more = clc_read(clc_resp, x, y, z);
            fence_proxy_async_smem();         // this read before the next response overwrites it
            if (more) w = fwd_item(a, x, y, z, group);
            item_slot[0] = make_int4(w.b, w.h, w.hi, w.two);
            item_slot[1] = make_int4(w.ns, w.lo, w.n, w.extra);
            item_slot[2] = make_int4(w.thin, more ? 1 : 0, 0, 0);
            mbar_arrive(item_full);
            ++items;
          }
        }
        if (!ok) report(a.status, kErrWindow + 1, w.hi, c);
      }
    } else if (warp == 1 && elect_one()) {
      const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0);
      const uint32_t idesc_pv = make_idesc_bf16(128, 128, 0, 1);
      const uint64_t dq = desc_kmajor(smem_u32(sQ), 0), dk = desc_kmajor(smem_u32(sK), 0);
      const uint64_t dv = desc_mnmajor(smem_u32(sV), 0);
      constexpr uint64_t kTileOff = (uint64_t)(kTile >> 4);
      uint32_t base = 0;              // K / V tiles of the items before this one
      uint32_t qc[2] = {0, 0}, pc[2] = {0, 0};
      bool ok = true, more = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code, uint32_t d) -> bool {
        if (mbar_wait(bar, parity, 8 * tmo)) {
          tc_fence_after_sync();
          return true;
        }
        report(a.status, kErrWindow + code, d, base);
        return false;
      };
      const uint32_t idesc_thin = make_idesc_bf16(128, kThinKeys, 0, 0);
      // Scores of tile t against entry x of the list.  The later tile that uses an entry gives its K back: tile 1 where both do.
      auto issue_s = [&](int t, int x) -> bool {
        const uint32_t at = base + x;
        if (!wait(k_full + (at & 1), (at >> 1) & 1, 3, t)) return false;
        const uint64_t dqt = dq + t * kTileOff, dkt = dk + (at & 1) * kTileOff;
        const uint32_t idesc = x == 0 && (w.thin >> t & 1) ? idesc_thin : idesc_s;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = (uint64_t)(((k >> 2) * kHalf + (k & 3) * 32) >> 4);
          umma_f16(tmem + t * 128, dqt + off, dkt + off, idesc, k != 0);
        }
        umma_commit(s_full + t);
        if (x == w.last(t)) umma_commit(q_empty + t);
        if (t == 1 || !w.uses(1, x)) umma_commit(k_empty + (at & 1));
        return true;
      };
      while (ok && more) {
        for (int t = 0; t < 1 + w.two && ok; ++t) {
          ok = wait(q_full + t, qc[t] & 1, 2, t);
          ++qc[t];
          if (ok) ok = issue_s(t, w.first(t));
        }
        for (int x = 0; x < w.n && ok; ++x) {
          const uint32_t at = base + x;
          if (!(ok = wait(v_full + (at & 1), (at >> 1) & 1, 4, 2))) break;
          const uint64_t dvs = dv + (at & 1) * kTileOff;
          for (int t = 0; t < 2; ++t) {
            if (!w.uses(t, x)) continue;
            const bool thin = x == 0 && (w.thin >> t & 1);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (ok) ok = wait(p_ready + 2 * t + half, pc[t] & 1, 4, t);
              if (ok) {
#pragma unroll
                for (int k = half * 6; k < 6 + half * 2; ++k)   // 16 bf16 of a row of P = 8 TMEM columns per step
                  if (k == 0 || !thin)
                    umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, dvs + (uint64_t)((k * 2048) >> 4), idesc_pv,
                                x != w.first(t) || k != 0);
              }
            }
            if (!ok) break;
            ++pc[t];
            if (t == 1 || !w.uses(1, x)) umma_commit(v_empty + (at & 1));
            if (x == w.last(t)) umma_commit(o_done + t);
            else if (!(ok = issue_s(t, w.next(t, x)))) break;
          }
        }
        if (ok) {
          base += w.n;
          more = next_item(w);
          mbar_arrive(clc_empty);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFwdRegsHigh));
    // ---------------- softmax / output: one thread per query row ----------------
    const int t = (warp >> 2) - 1;            // this warpgroup's tile
    const int q4 = warp & 3;
    const int row = q4 * 32 + lane;           // row inside the tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(q4 * 32) << 16;
    const uint32_t ts = tmem + t * 128 + lane_off, to = tmem + 256 + t * 128 + lane_off;
    const float sl2 = a.scale * kLog2e;
    const uint64_t sl2x2 = f32x2(sl2, sl2);
    uint8_t* stage = sO + (warp - 4) * kFwdWarpStage;
    uint32_t sc = 0, oc = 0;                  // S tiles / outputs of this tile so far
    bool ok = true, more = true;
    FwdItem w = fwd_item(a, blockIdx.x, blockIdx.y, blockIdx.z, group);
    while (more) {
      const bool live = t == 0 || w.two;
      const int i_blk = w.hi - t, query = i_blk * kBlk + row;
      float m_used = -INFINITY, l = 0.f;
      bool first = true;
      for (int x = 0; x < w.n && live; ++x) {
        if (!w.uses(t, x)) continue;
        if (!warp_wait(s_full + t, sc & 1, 8 * tmo)) {
          if (lane == 0) report(a.status, kErrWindow + 5, x, t);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        ++sc;
        if (x == 0 && (w.thin >> t & 1)) {
          // nothing but the first tokens, which the whole tile sees
          uint32_t r[16], pk[8];
          tmem_ld_32x16(ts, r);
          tmem_ld_wait();
          float m = -INFINITY;
#pragma unroll
          for (int i = 0; i < kThinKeys; ++i) {
            if (i >= a.sinks) r[i] = 0xff800000u;
            m = fmaxf(m, __uint_as_float(r[i]));
          }
          first = false;
          m_used = m * sl2;
          const float m_here = m_used == -INFINITY ? 0.f : m_used;
#pragma unroll
          for (int i = 0; i < kThinKeys; i += 2) {
            const float x0 = fast_exp2(fmaf(__uint_as_float(r[i]), sl2, -m_here)), x1 = fast_exp2(fmaf(__uint_as_float(r[i + 1]), sl2, -m_here));
            l += x0 + x1;
            pk[i >> 1] = pack_bf16(x0, x1);
          }
          tmem_st_32x8(ts, pk);
          tmem_st_wait();
          tc_fence_before_sync();
          mbar_arrive(p_ready + 2 * t);
          mbar_arrive(p_ready + 2 * t + 1);
          continue;
        }
        const int key0 = w.block(x) * kBlk;
        // only blocks on the diagonal and on the window's edge, and far ones with first tokens, carry mask arithmetic
        const bool masked = key0 == i_blk * kBlk || (i_blk * kBlk + kBlk - 1 - key0 >= a.window && key0 + kBlk > a.sinks);
        uint32_t r[4][32];
        float mc[4];
        // the whole row with one wait: four loads in flight
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(ts + c * 32, r[c]);
        tmem_ld_wait();
        if (masked) {
          const int below = query - key0 + 1;                          // keys of this block up to the query
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t seen = low_bits(below - c * 32) & (~low_bits(below - a.window - c * 32) | low_bits(a.sinks - key0 - c * 32));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(seen >> i & 1)) r[c][i] = 0xff800000u;             // -inf
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float m0 = __uint_as_float(r[c][0]), m1 = __uint_as_float(r[c][1]);
#pragma unroll
          for (int i = 2; i + 3 < 32; i += 4) {
            m0 = max3(m0, __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
            m1 = max3(m1, __uint_as_float(r[c][i + 2]), __uint_as_float(r[c][i + 3]));
          }
          mc[c] = max3(fmaxf(m0, m1), __uint_as_float(r[c][30]), __uint_as_float(r[c][31]));
        }
        const float m_blk = fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])) * sl2;
        if (first) {
          first = false;
          m_used = m_blk;
        } else {
          // these scores are complete, hence the P V before them is too: O may be rescaled in place
          const float m_new = fmaxf(m_used, m_blk);
          const bool need = (m_new - m_used) > 8.0f;
          if (__any_sync(0xffffffffu, need)) {
            const float alpha = need ? exp2f(m_used - m_new) : 1.0f;
            if (need) {
              l *= alpha;
              m_used = m_new;
            }
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld_32x32(to + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32(to + c * 32, o);
            }
          }
        }
        // (a row that has seen nothing yet: all its scores are -inf, and -inf - 0 gives the probability 0 that -inf + inf would not)
        const float m_here = m_used == -INFINITY ? 0.f : m_used;
        const uint64_t neg_m = f32x2(-m_here, -m_here);
        uint64_t sum[4];
        auto add_quarter = [&](int c) {
          sum[c] = f32x2(__uint_as_float(r[c][0]), __uint_as_float(r[c][1]));
#pragma unroll
          for (int i = 2; i < 32; i += 2)
            sum[c] = add2(sum[c], f32x2(__uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1])));
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            split(fma2(f32x2(__uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1])), sl2x2, neg_m), x0, x1);
            x0 = fast_exp2(x0);
            x1 = fast_exp2(x1);
            r[c][i] = __float_as_uint(x0);
            r[c][i + 1] = __float_as_uint(x1);
            pk[i >> 1] = pack_bf16(x0, x1);
          }
          // P columns [32c, 32c+32) as bf16 = TMEM columns [16c, 16c+16): over S columns already read
          tmem_st_32x16(ts + c * 16, pk);
          if (c < 2) add_quarter(c);
          if (c >= 2) {
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive(p_ready + 2 * t + c - 2);
          }
        }
        // the row's sum; its second half is off the chain that the products wait for
        add_quarter(2);
        add_quarter(3);
        float s0, s1;
        split(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
        l += s0 + s1;
      }
      if (ok && live) {
        if (!warp_wait(o_done + t, oc & 1, 8 * tmo)) {
          if (lane == 0) report(a.status, kErrWindow + 7, t, 0);
          ok = false;
        }
        ++oc;
      }
      if (!ok) break;
      if (live) {
        tc_fence_after_sync();
        const float inv = 1.0f / l;
        // The warp's 32 rows leave through shared memory, 64 columns at a time, as TMA stores: nothing here waits for
        // the memory system (with plain stores a warp stalls when all SMs write their items at the same time).
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t o[2][32];
          tmem_ld_32x32(to + half * 64, o[0]);
          tmem_ld_32x32(to + half * 64 + 32, o[1]);
          warp_stage_free();
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 u;
              u.x = pack_bf16(__uint_as_float(o[c][q * 8 + 0]) * inv, __uint_as_float(o[c][q * 8 + 1]) * inv);
              u.y = pack_bf16(__uint_as_float(o[c][q * 8 + 2]) * inv, __uint_as_float(o[c][q * 8 + 3]) * inv);
              u.z = pack_bf16(__uint_as_float(o[c][q * 8 + 4]) * inv, __uint_as_float(o[c][q * 8 + 5]) * inv);
              u.w = pack_bf16(__uint_as_float(o[c][q * 8 + 6]) * inv, __uint_as_float(o[c][q * 8 + 7]) * inv);
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((c * 4 + q) ^ (lane & 7)) << 4)) = u;   // 128-byte swizzle
            }
          warp_store_box(&tm_out, stage, w.h * kD + half * 64, i_blk * kBlk + q4 * 32, w.b, a.seq);
        }
        if (query < a.seq) a.lse[((int64_t)w.b * a.heads + w.h) * a.seq + query] = m_used * kLn2 + logf(l);
      }
      more = next_item(w);
      __syncwarp();                              // every lane has read the slot
      if (lane == 0) mbar_arrive(clc_empty);
    }
    if (lane == 0) bulk_wait_all<0>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ==========================================================================================
// backward
// ==========================================================================================
// delta[b, h, s] = -rowsum(dO * O) * scale and lse2[b, h, s] = -lse * log2(e), of sequences padded to whole tiles: rows beyond the end
// get 0 and -inf, so that their probabilities are 0.  16 lanes with a 16-byte vector each take one head of kDeltaRows tokens.
constexpr int kDeltaRows = 4;
__global__ void __launch_bounds__(256)
window_delta_kernel(const uint4* out, const uint4* dout, float* delta, uint32_t groups, uint32_t seq, uint32_t padded,
                    uint32_t heads, const float* lse, float* lse2, float scale) {
  grid_wait();
  grid_trigger();
  const uint32_t sub = threadIdx.x & 15;
  const uint32_t w = blockIdx.x * (blockDim.x >> 4) + (threadIdx.x >> 4);   // (sequence, group of tokens, head)
  const uint32_t tg = w / heads, h = w - tg * heads, per = padded / kDeltaRows, b = tg / per, s0 = (tg - b * per) * kDeltaRows;
  uint4 o[kDeltaRows], d[kDeltaRows];
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    o[i] = d[i] = make_uint4(0u, 0u, 0u, 0u);
    if (w < groups && s0 + i < seq) {
      const int64_t at = (((int64_t)b * seq + s0 + i) * heads + h) * 16 + sub;
      o[i] = ld_stream(out + at);
      d[i] = ld_stream(dout + at);
    }
  }
  float mine = 0.f;                      // the sum of row `sub`
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    const uint32_t ov[4] = {o[i].x, o[i].y, o[i].z, o[i].w}, dv[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      s += __uint_as_float(ov[k] << 16) * __uint_as_float(dv[k] << 16) +
           __uint_as_float(ov[k] & 0xffff0000u) * __uint_as_float(dv[k] & 0xffff0000u);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (sub == i) mine = s;
  }
  if (w < groups && sub < kDeltaRows) {
    const int64_t row = (int64_t)b * heads + h;
    const uint32_t s = s0 + sub;
    delta[row * padded + s] = -mine * scale;
    lse2[row * padded + s] = s < seq ? -lse[row * seq + s] * kLog2e : -INFINITY;
  }
}

// Few first tokens (up to kThinKeys) beyond the window: what far queries add to their dK and dV comes from here, with the row sums, so that
// no key-major item streams a whole sequence for a handful of keys.  Queries come in tiles of 16 rows, a warp's ring filled by itself
// (cp.async); the first tokens are the 8 (or twice 8) columns of matrix fragments: S = Q K^T and dP = dO V^T, then dV^T += dO^T P and
// dK^T += Q^T dS, whose B operands are the score fragments transposed.  A CTA takes a run of the tiles of one key head (of all query
// heads that share it) and leaves its sums in `parts`; the key-major item of block 0 adds their sum before it rounds.  mma.sync: 32
// instructions a tile of 8 or 12 KiB and 8 first tokens.
// It reads O, dO and, of far queries, Q once: 186 MB in 43 us with cold caches (4 x 2048, 32 heads, window 512), 55 % of DRAM where a copy reaches 85.
constexpr int kRowsWarps = 4, kRowsStages = 2, kRowsTile = 16 * kD * 2;
constexpr int kRowsSmem = kRowsWarps * kRowsStages * 3 * kRowsTile;
constexpr int kRowsPart = 2 * kThinKeys * kD;      // floats of a CTA: dV, dK
static_assert(kRowsWarps * kRowsPart * 4 <= kRowsSmem, "the warps' sums take the place of the tiles");
struct RowsArgs {
  const __nv_bfloat16 *qkv, *out, *dout;
  const float* lse;
  float *lse2, *delta, *parts;
  int seq, padded, kv, group, window, sinks, per;   // per: tiles of a CTA
  float scale;
};
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
// kCols: groups of 8 first tokens.
template <int kCols>
__global__ void __launch_bounds__(kRowsWarps * 32, 2)
window_rows_kernel(const __grid_constant__ RowsArgs a) {
  extern __shared__ __align__(128) uint8_t rows_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y / a.kv, h = blockIdx.y - b * a.kv, heads = a.kv * a.group, width = a.kv * (a.group + 2) * kD;
  const int per_head = a.padded / 16, t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.group * per_head);
  const uint32_t ring = smem_u32(rows_smem) + warp * kRowsStages * 3 * kRowsTile;
  const __nv_bfloat16* first = a.qkv + (int64_t)b * a.seq * width + h * (a.group + 2) * kD;   // row 0, query head 0 of this key head
  grid_trigger();
  grid_wait();
  // chunk c of row r of a tile lies at c ^ (r % 8): fragments are read without conflicts
  auto fetch = [&](int t, int stage) {
    if (t < t1) {
      const int m = t / per_head, q0 = (t - m * per_head) * 16;
      const bool far = q0 + 15 >= a.window;
      const uint32_t at = ring + stage * 3 * kRowsTile;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 2 + (lane >> 4), c = lane & 15;
        const bool there = q0 + r < a.seq;
        const int64_t tok = there ? q0 + r : 0;
        const int64_t o = (((int64_t)b * a.seq + tok) * heads + h * a.group + m) * kD + c * 8;
        const uint32_t to = at + r * 256 + ((c ^ (r & 7)) << 4);
        copy16(to, a.out + o, there);
        copy16(to + kRowsTile, a.dout + o, there);
        if (far) copy16(to + 2 * kRowsTile, first + tok * width + m * kD + c * 8, there);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(t0 + warp, 0);
  // first tokens as B fragments: column lane / 4 of each 8, rows (features) 2 (lane % 4) and + 8 of each 16
  uint32_t kb[kCols][8][2], vb[kCols][8][2];
#pragma unroll
  for (int n = 0; n < kCols; ++n)
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = n * 8 + (lane >> 2), col = ks * 16 + i * 8 + (lane & 3) * 2;
        const __nv_bfloat16* k = first + (int64_t)key * width + a.group * kD + col;
        kb[n][ks][i] = key < a.sinks ? *reinterpret_cast<const uint32_t*>(k) : 0u;
        vb[n][ks][i] = key < a.sinks ? *reinterpret_cast<const uint32_t*>(k + kD) : 0u;
      }
  float dv[kCols][8][4] = {}, dk[kCols][8][4] = {};   // [features of 16][first tokens of 8]
  const float sl2 = a.scale * kLog2e;
  int stage = 0;
  for (int t = t0 + warp; t < t1; t += kRowsWarps) {
    fetch(t + kRowsWarps, stage ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint32_t to = ring + stage * 3 * kRowsTile, td = to + kRowsTile, tq = td + kRowsTile;
    const int m = t / per_head, q0 = (t - m * per_head) * 16;
    const int64_t head = (int64_t)b * heads + h * a.group + m;
    // row sums: two lanes a row, whose chunks are taken in orders that do not meet in a bank
    float mine = 0.f;
    {
      const int r = lane >> 1, half = lane & 1, q = q0 + r;
      const float lse = q < a.seq ? a.lse[head * a.seq + q] : INFINITY;
      const uint8_t* row = rows_smem + (to - smem_u32(rows_smem)) + r * 256;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = (half * 8 + (i ^ (half * 4))) ^ (r & 7);
        const uint4 o = *reinterpret_cast<const uint4*>(row + c * 16), d = *reinterpret_cast<const uint4*>(row + kRowsTile + c * 16);
        const uint32_t ov[4] = {o.x, o.y, o.z, o.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mine += __uint_as_float(ov[k] << 16) * __uint_as_float(dd[k] << 16) +
                  __uint_as_float(ov[k] & 0xffff0000u) * __uint_as_float(dd[k] & 0xffff0000u);
      }
      mine += __shfl_xor_sync(0xffffffffu, mine, 1);
      mine = half ? -lse * kLog2e : -mine * a.scale;               // (beyond the end: -inf, 0)
      (half ? a.lse2 : a.delta)[head * a.padded + q] = mine;
    }
    if (q0 + 15 >= a.window) {
      float s[kCols][4] = {}, dp[kCols][4] = {};
      const int r = lane & 15;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t x[4];
        const uint32_t at = r * 256 + (((ks * 2 + (lane >> 4)) ^ (r & 7)) << 4);
        load4(x, tq + at);
#pragma unroll
        for (int n = 0; n < kCols; ++n) mma(s[n], x, kb[n][ks][0], kb[n][ks][1]);
        load4(x, td + at);
#pragma unroll
        for (int n = 0; n < kCols; ++n) mma(dp[n], x, vb[n][ks][0], vb[n][ks][1]);
      }
      uint32_t p[kCols][2], g[kCols][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = (lane >> 2) + i * 8;
        const float delta = __shfl_sync(0xffffffffu, mine, 2 * q), lse2 = __shfl_sync(0xffffffffu, mine, 2 * q + 1);
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
          float e[2], d[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int key = n * 8 + (lane & 3) * 2 + j;
            // (a query beyond the end is zeros, whose score for an infinite key is NaN)
            const bool seen = key < a.sinks && q0 + q - key >= a.window && q0 + q < a.seq;
            e[j] = seen ? fast_exp2(fmaf(s[n][i * 2 + j], sl2, lse2)) : 0.f;
            d[j] = seen ? e[j] * fmaf(dp[n][i * 2 + j], a.scale, delta) : 0.f;
          }
          p[n][i] = transpose8(pack_bf16(e[0], e[1]));
          g[n][i] = transpose8(pack_bf16(d[0], d[1]));
        }
      }
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        // 16 features of the 16 queries, transposed: rows 0-7 and 8-15 of the fragment are features, its columns queries
        uint32_t x[4];
        const int q = (lane & 7) + (lane >> 4) * 8;
        const uint32_t at = q * 256 + (((f * 2 + (lane >> 3 & 1)) ^ (q & 7)) << 4);
        load4_trans(x, td + at);
#pragma unroll
        for (int n = 0; n < kCols; ++n) mma(dv[n][f], x, p[n][0], p[n][1]);
        load4_trans(x, tq + at);
#pragma unroll
        for (int n = 0; n < kCols; ++n) mma(dk[n][f], x, g[n][0], g[n][1]);
      }
    }
    __syncwarp();                                  // the stage has been read
    stage ^= 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* sums = reinterpret_cast<float*>(rows_smem) + warp * kRowsPart;
#pragma unroll
  for (int n = 0; n < kCols; ++n)
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* at = sums + (n * 8 + (lane & 3) * 2 + (i & 1)) * kD + f * 16 + (lane >> 2) + (i >> 1) * 8;
        at[0] = dv[n][f][i];
        at[kThinKeys * kD] = dk[n][f][i];
      }
  __syncthreads();
  float* part = a.parts + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kRowsPart;
  for (int i = threadIdx.x; i < kRowsPart; i += kRowsWarps * 32) {
    float v = 0.f;
    if ((i / kD) % kThinKeys < kCols * 8)
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) v += reinterpret_cast<const float*>(rows_smem)[w * kRowsPart + i];
    part[i] = v;
  }
}

// The CTAs' sums of each key head, added up in their order: a key-major item that added them itself would wait for memory once for each.
__global__ void __launch_bounds__(128)
window_parts_kernel(const float* parts, float* sums, int chunks) {
  grid_trigger();
  grid_wait();
  const int64_t at = blockIdx.x * 128 + threadIdx.x;
  const float* p = parts + (int64_t)blockIdx.y * chunks * kRowsPart + at;
  float v = 0.f;
#pragma unroll 8
  for (int c = 0; c < chunks; ++c) v += p[(int64_t)c * kRowsPart];
  sums[(int64_t)blockIdx.y * kRowsPart + at] = v;
}

// Key-major items accumulate dV and dK of 128 keys over the query blocks that see them, of every head of the group; query-major
// items dQ of 128 queries over their list of key blocks.  Roles, rings and tensor memory as in attn_bwd2_kernel.  P (for dV) and dS
// are rounded to bf16 as operands; dS is formed from P in fp32.
// What bounds it: a key-major pair takes 2650 cycles (2048 of products), an item about 5000 more in which its output leaves and the next
// one's tiles arrive (30 % of that pass at a window of 512); over long runs the power cap (1.5 GHz), which gives back in clock about half of
// what a cycle saved brings.
// 4 x 2048, 32 heads, window 512, 4 first tokens: 300 us (key-major 150, query-major 110, row sums and first tokens 37; first tokens in items of
// their own kind 327); 2 x 5003, 16 heads on 4, window 1000, 16 first tokens: 270 (418).
constexpr int kBwdPoly = 2;                 // key-major: exponentials of every eight that run on the FMA pipe
constexpr int kBwdWarps = 16;               // element-wise warps
constexpr int kBwdCols = kBlk * 4 / kBwdWarps;   // columns of a row per element-wise thread
constexpr int kBwdStage = 32 * kBwdCols * 2;     // output staging per element-wise warp
constexpr int kStatBytes = kBlk * 4;        // lse2 or delta of 128 queries
constexpr int kThinBytes = kThinKeys * kD * 2;
constexpr int kBwdAlignSlack = 192;
constexpr size_t kBwdBars = 7 * kTile + 5 * kStatBytes;   // where the barriers are
constexpr size_t kBwdSmem = kBwdBars + 320 + kBwdAlignSlack;
static_assert(kBwdWarps * kBwdStage == kTile, "an item's staged output takes the place of a tile");
static_assert(kBwdSmem <= 232448, "shared memory of a CTA");
constexpr int kBwdThreads = 96 + 32 * kBwdWarps;

struct WinBwdArgs {
  const float* lse2;    // -lse * log2(e)          (written by window_delta_kernel)
  const float* delta;   // -rowsum(dO * O) * scale (written by window_delta_kernel)
  uint32_t items;       // item i < items is key-major, items + i query-major
  int key_group, query_group;   // rows of items (sequence, head) that are dealt together
  int batch, seq, kv, group, heads, window, sinks;
  int key_sinks;        // first tokens whose keys key-major items stream every later query for: none of the few (`far` has them)
  const float* far;     // [batch * kv][dV, dK][kThinKeys][128] of the few, or null
  float scale;
  uint32_t* status;
  uint64_t timeout_ns;
};
__device__ __forceinline__ int64_t stat_at(const WinBwdArgs& a, int b, int h, int blk) {
  const int nblk = (a.seq + kBlk - 1) / kBlk;
  return (((int64_t)b * a.heads + h) * nblk + blk) * kBlk;
}

struct BwdItem {
  int b, h, blk, n_it;  // sequence, key head (key-major) or query head, owned block, streamed blocks
  int i0, per;          // key-major: first query block, query blocks of a head; query-major: blocks with first tokens, first of the window
  int kv;               // key head
  int flags;            // kMore: there is such an item; kThin: query-major, the first block streams no more than its kThinKeys first tokens
};
enum { kMore = 1, kThin = 2 };
static_assert(sizeof(BwdItem) == 32, "two vectors");
// The streamed blocks of an item one after another.
template <bool kKeyMajor>
struct Streamed {
  int h, blk;           // query head and block
  __device__ __forceinline__ Streamed(const WinBwdArgs& a, const BwdItem& w)
      : h(kKeyMajor ? w.h * a.group : w.h), blk(kKeyMajor ? w.i0 : w.i0 > 0 ? 0 : w.per) {}
  __device__ __forceinline__ void next(const BwdItem& w) {
    ++blk;
    if (kKeyMajor) {
      if (blk == w.i0 + w.per) {
        blk = w.i0;
        ++h;
      }
    } else if (blk == w.i0) {
      blk = w.per;
    }
  }
};
// kThinItems: few first tokens are streamed alone (not by the kernel of both kinds, which has no registers left for it).
template <bool kKeyMajor, bool kThinItems>
__device__ __forceinline__ BwdItem bwd_item(const WinBwdArgs& a, uint32_t item) {
  BwdItem w;
  const int nblk = (a.seq + kBlk - 1) / kBlk, group = kKeyMajor ? a.key_group : a.query_group, heads = kKeyMajor ? a.kv : a.heads;
  const uint32_t i = kKeyMajor ? item : item - a.items, row = i / (uint32_t)group;
  const int bh = (int)(row / (uint32_t)nblk) * group + (int)(i - row * (uint32_t)group), y = (int)(row % (uint32_t)nblk);
  w.b = bh / heads;
  w.h = bh - w.b * heads;
  // the longest items of a group first: key block 0, the last query block
  w.blk = kKeyMajor ? y : nblk - 1 - y;
  if (kKeyMajor) {
    const int last = w.blk * kBlk < a.key_sinks ? nblk - 1 : min(nblk - 1, (w.blk * kBlk + kBlk - 1 + a.window - 1) / kBlk);
    w.i0 = w.blk;
    w.per = last - w.blk + 1;
    w.n_it = w.per * a.group;
  } else {
    w.i0 = min(sink_blocks(a), w.blk + 1);
    w.per = max(w.i0, window_block(a, w.blk));
    w.n_it = w.i0 + max(0, w.blk + 1 - w.per);
  }
  w.kv = kKeyMajor ? w.h : w.h / a.group;
  w.flags = kMore | (kThinItems && w.i0 == 1 && a.far != nullptr && window_block(a, w.blk) > 0 ? kThin : 0);
  return w;
}

// How many of the distances 8 t + (0 or 1), t = -3 .. 3, are below d.
__device__ __forceinline__ int below(int d) { return d <= -24 ? 0 : ((d + 24) >> 3) * 2 + min((d + 24) & 7, 2); }

// A CTA's run of items of one kind, from `item` on, until cluster launch control has none left or one of the other kind (the
// response stays in shared memory).  False after a timeout.  At its end every copy and every tcgen05 operation has arrived
// where it was announced, so the barriers can be set up anew for the next run.
// kKeyMajor = true:  resident tiles K, V (this item's 128 keys), streamed Q, dO; accumulators dV, dK.
//                    TMEM lanes = keys, columns = queries: lse / delta vary along the columns.
// kKeyMajor = false: resident tiles Q, dO (this item's 128 queries), streamed K, V; accumulator dQ.
//                    TMEM lanes = queries, columns = keys: lse / delta are per thread.
template <bool kKeyMajor, bool kThinItems>
__device__ __forceinline__ bool window_bwd_run(const CUtensorMap& tm_qkv, const CUtensorMap& tm_do, const CUtensorMap& tm_dqkv,
                                               const CUtensorMap& tm_thin,
                                              const WinBwdArgs& a, uint8_t* smem, uint32_t tmem, uint32_t item) {
  uint8_t* sR0 = smem;                      // resident: K (key-major) or Q
  uint8_t* sR1 = smem + kTile;              // resident: V (key-major) or dO
  // Streamed tiles, a ring each.  Q / K is read by the first and the last product of a block, dO (key-major) by the
  // second and third, V (query-major) by the second alone.
  constexpr uint32_t kRing0 = 3, kRing1 = 2;
  uint8_t* sS0 = smem + 2 * kTile;          // Q or K
  uint8_t* sS1 = smem + 5 * kTile;          // dO or V; between items the stage of an item's last block takes its output
  // key-major: lse2 travels with Q, delta with dO.  delta(i+2) takes the slot of delta(i): its producer waits for dS(i).
  float* sLse = reinterpret_cast<float*>(smem + 7 * kTile);   // [3][128]
  float* sDelta = sLse + 3 * kBlk;                            // [2][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBwdBars);   // 30 is the tensor-memory address
  uint8_t* clc_resp = reinterpret_cast<uint8_t*>(bars);   // 16 bytes
  uint64_t* clc_full = bars + 2;
  uint64_t* clc_empty = bars + 3;
  uint64_t* res_full = bars + 4;            // [2] resident tiles: the one that S reads, the one that dP reads
  uint64_t* res_empty = bars + 6;           // [2]
  uint64_t* full0 = bars + 8;               // [3] rings
  uint64_t* empty0 = bars + 11;             // [3]
  uint64_t* full1 = bars + 14;              // [2]
  uint64_t* empty1 = bars + 16;             // [2]
  uint64_t* s_full = bars + 18;
  uint64_t* s_free = bars + 19;             // query-major: S is in registers
  uint64_t* dp_full = bars + 20;            // [2] (key-major uses [0] only)
  uint64_t* ds_ready = bars + 22;           // [2] dS is in TMEM, even and odd blocks
  uint64_t* p_ready = bars + 24;            // [2] key-major: the first / second 16 columns of every warp's P^T
  uint64_t* acc_done = bars + 26;           // [2] key-major: dV / dK; query-major: [1] dQ
  uint64_t* out_read = bars + 28;           // [2] the copy engine has read the output staged in a stage of ring 1
  uint64_t* item_full = bars + 31;          // the next item, as the producer of ring 0 has worked it out
  uint64_t* out_read0 = bars + 32;          // [3] key-major: as out_read, of ring 0
  int4* item_slot = reinterpret_cast<int4*>(bars + 36);   // [2]

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint64_t tmo = a.timeout_ns;

  if (threadIdx.x == 0) {
    mbar_init(clc_full, 1);
    mbar_init(item_full, 1);
    mbar_init(clc_empty, 2 + kBwdWarps);    // producer of ring 1 and MMA thread, element-wise warps
    for (int i = 0; i < 3; ++i) {
      mbar_init(full0 + i, 1);
      mbar_init(empty0 + i, 1);
      mbar_init(out_read0 + i, kBwdWarps);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, kBwdWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(res_full + i, 1);
      mbar_init(res_empty + i, 1);
      mbar_init(full1 + i, 1);
      mbar_init(empty1 + i, 1);
      mbar_init(dp_full + i, 1);
      mbar_init(ds_ready + i, kBwdWarps);
      mbar_init(p_ready + i, kBwdWarps);
      mbar_init(acc_done + i, 1);
      mbar_init(out_read + i, kBwdWarps);
    }
    mbar_fence_init();
  }
  __syncthreads();
  // key-major:   S^T [0,128)  dP^T [128,256)  dV [256,384)  dK [384,512)
  // query-major: S [0,128)  dP buffers [128,256) [256,384)  dQ [384,512)
  const uint32_t t_dp = tmem + 128;
  const auto dp_buf = [](uint32_t q) -> uint32_t { return kKeyMajor ? 0 : q & 1; };         // of streamed block q
  const auto dp_phase = [](uint32_t q) -> uint32_t { return (kKeyMajor ? q : q >> 1) & 1; };
  const uint32_t t_acc0 = tmem + (kKeyMajor ? 256 : 384), t_acc1 = tmem + 384;

  BwdItem w = bwd_item<kKeyMajor, kThinItems>(a, item);
  bool ok = true;
  // The next item, which the producer of ring 0 has worked out for all: false when there is none of this kind (or on a timeout).
  uint32_t items = 0;                       // items finished by this thread
  auto next_item = [&]() -> bool {
    if (!mbar_wait(item_full, items & 1, 8 * tmo)) {
      report(a.status, kErrWindow + 18, items, 0);
      ok = false;
      return false;
    }
    ++items;
    const int4 lo = item_slot[0], hi = item_slot[1];
    if (hi.w == 0) return false;
    w.flags = hi.w;
    w.b = lo.x; w.h = lo.y; w.blk = lo.z; w.n_it = lo.w;
    w.i0 = hi.x; w.per = hi.y; w.kv = hi.z;
    return true;
  };
  uint32_t g = 0;                           // streamed blocks so far: stages and phases of the rings and the hand-overs

  if (warp == 0) {
    // resident tile of S, ring of Q or K, next items
    if (elect_one()) {
      bool more = true;
      uint32_t outs[3] = {0, 0, 0};           // key-major: outputs staged in each stage so far
      bool staged[3] = {false, false, false}; // the last user of the stage was an item's output
      while (ok && more) {
        // the resident tile of S first, then the item's first streamed tile: S needs no more
        if (!(ok = mbar_wait(res_empty, (items & 1) ^ 1, 8 * tmo))) break;
        mbar_expect_tx(res_full, kTile);
        load_tile(sR0, &tm_qkv, res_full, kKeyMajor ? col_k(a, w.h) : col_q(a, w.kv, w.h), w.blk * kBlk, w.b);           // K or Q
        Streamed<kKeyMajor> s(a, w);
        for (int it = 0; it < w.n_it && ok; ++it, ++g, s.next(w)) {
          const uint32_t st = g % kRing0;
          if (!(ok = mbar_wait(empty0 + st, ((g / kRing0) & 1) ^ 1, 8 * tmo))) break;
          if (kKeyMajor && staged[st] && !(ok = mbar_wait(out_read0 + st, (outs[st] - 1) & 1, 8 * tmo))) break;
          staged[st] = false;
          const bool thin = kThinItems && it == 0 && (w.flags & kThin);
          mbar_expect_tx(full0 + st, thin ? kThinBytes : kTile + (kKeyMajor ? kStatBytes : 0));
          load_tile(sS0 + st * kTile, thin ? &tm_thin : &tm_qkv, full0 + st, kKeyMajor ? col_q(a, w.h, s.h) : col_k(a, w.kv), s.blk * kBlk, w.b);
          if (kKeyMajor) bulk_g2s(sLse + st * kBlk, a.lse2 + stat_at(a, w.b, s.h, s.blk), kStatBytes, full0 + st);
        }
        if (ok) {
          const uint32_t st = (g - 1) % kRing0;
          staged[st] = kKeyMajor;
          ++outs[st];
        }
        // every thread has the item that the slot holds: ask for the next and work it out
        if (ok && (ok = mbar_wait(clc_empty, (items & 1) ^ 1, 8 * tmo))) {
          mbar_expect_tx(clc_full, 16);
          clc_try_cancel(clc_resp, clc_full);
          uint32_t x, y, z;
          if ((ok = mbar_wait(clc_full, items & 1, 8 * tmo))) {
            more = clc_read(clc_resp, x, y, z) && (x < a.items) == kKeyMajor;
            fence_proxy_async_smem();         // this read before the next response overwrites it
            if (more) w = bwd_item<kKeyMajor, kThinItems>(a, x);
            item_slot[0] = make_int4(w.b, w.h, w.blk, w.n_it);
            item_slot[1] = make_int4(w.i0, w.per, w.kv, more ? w.flags : 0);
            mbar_arrive(item_full);
            ++items;
          }
        }
      }
      // what is still under way (a timeout above is reported here too)
      for (uint32_t q = g; q < g + kRing0 && ok; ++q) ok = mbar_wait(empty0 + q % kRing0, ((q / kRing0) & 1) ^ 1, 8 * tmo);
      ok = ok && mbar_wait(res_empty, (items & 1) ^ 1, 8 * tmo);
      if (!ok) report(a.status, kErrWindow + 11, w.blk, g);
    }
  } else if (warp == 2 + kBwdWarps) {
    // resident tile of dP, ring of dO or V: by a thread of its own, because a stage of one ring is often free long before one of the other
    if (elect_one()) {
      bool more = true;
      uint32_t outs[2] = {0, 0};              // outputs staged in either stage so far
      bool staged[2] = {false, false};        // the last user of the stage was an item's output
      while (ok && more) {
        if ((ok = mbar_wait(res_empty + 1, (items & 1) ^ 1, 8 * tmo))) {
          mbar_expect_tx(res_full + 1, kTile);
          if (kKeyMajor) load_tile(sR1, &tm_qkv, res_full + 1, col_k(a, w.h) + kD, w.blk * kBlk, w.b);     // V
          else load_tile(sR1, &tm_do, res_full + 1, w.h * kD, w.blk * kBlk, w.b);                            // dO
        }
        Streamed<kKeyMajor> s(a, w);
        for (int it = 0; it < w.n_it && ok; ++it, ++g, s.next(w)) {
          const uint32_t st = g % kRing1;
          if (!(ok = mbar_wait(empty1 + st, ((g / kRing1) & 1) ^ 1, 8 * tmo))) break;
          if (staged[st] && !(ok = mbar_wait(out_read + st, (outs[st] - 1) & 1, 8 * tmo))) break;
          staged[st] = false;
          const bool thin = kThinItems && it == 0 && (w.flags & kThin);
          mbar_expect_tx(full1 + st, thin ? kThinBytes : kTile + (kKeyMajor ? kStatBytes : 0));
          if (kKeyMajor) {
            load_tile(sS1 + st * kTile, &tm_do, full1 + st, s.h * kD, s.blk * kBlk, w.b);                                // dO
            if (g > 1 && !(ok = mbar_wait(ds_ready + st, ((g - 2) >> 1) & 1, 8 * tmo))) break;
            bulk_g2s(sDelta + st * kBlk, a.delta + stat_at(a, w.b, s.h, s.blk), kStatBytes, full1 + st);
          } else {
            load_tile(sS1 + st * kTile, thin ? &tm_thin : &tm_qkv, full1 + st, col_k(a, w.kv) + kD, s.blk * kBlk, w.b);                  // V
          }
        }
        if (ok) {
          const uint32_t st = (g - 1) % kRing1;
          staged[st] = true;
          ++outs[st];
        }
        if (ok) {
          more = next_item();
          mbar_arrive(clc_empty);
        }
      }
      for (uint32_t q = g; q < g + kRing1 && ok; ++q) ok = mbar_wait(empty1 + q % kRing1, ((q / kRing1) & 1) ^ 1, 8 * tmo);
      ok = ok && mbar_wait(res_empty + 1, (items & 1) ^ 1, 8 * tmo);
      if (!ok) report(a.status, kErrWindow + 11, w.blk, g);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t id_s = make_idesc_bf16(128, 128, 0, 0);      // A K-major (smem) * B K-major
      const uint32_t id_g = make_idesc_bf16(128, 128, 0, 1);      // A (TMEM) * B MN-major
      // descriptors of the first k-step of each operand; the others are these plus constants
      const uint64_t dr0 = desc_kmajor(smem_u32(sR0), 0), dr1 = desc_kmajor(smem_u32(sR1), 0);
      const uint64_t ds0k = desc_kmajor(smem_u32(sS0), 0), ds1k = desc_kmajor(smem_u32(sS1), 0);
      const uint64_t ds0m = desc_mnmajor(smem_u32(sS0), 0), ds1m = desc_mnmajor(smem_u32(sS1), 0);
      constexpr uint64_t kStageOff = (uint64_t)(kTile >> 4);
      bool more = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) -> bool {
        if (mbar_wait(bar, parity, 8 * tmo)) {
          tc_fence_after_sync();
          return true;
        }
        report(a.status, kErrWindow + code, g, items);
        return false;
      };
      // S (or S^T) / dP (or dP^T) of streamed block number q, once its tile is there and the block before is out of S (key-major:
      // the products that read its P^T were issued before)
      const uint32_t id_thin = make_idesc_bf16(128, kThinKeys, 0, 0);
      auto issue_s = [&](uint32_t q, uint32_t id_s) -> bool {
        const uint32_t st = q % kRing0;
        if (!kKeyMajor && q > 0 && !wait(s_free, (q - 1) & 1, 19)) return false;
        if (!wait(full0 + st, (q / kRing0) & 1, 13)) return false;
        const uint64_t tile = ds0k + st * kStageOff;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = (uint64_t)(((k >> 2) * kHalf + (k & 3) * 32) >> 4);
          umma_f16(tmem, dr0 + off, tile + off, id_s, k != 0);
        }
        umma_commit(s_full);
        return true;
      };
      auto issue_dp = [&](uint32_t q, uint32_t id_s) -> bool {
        const uint32_t st = q % kRing1;
        if (!wait(full1 + st, (q / kRing1) & 1, 13)) return false;
        const uint64_t tile = ds1k + st * kStageOff;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = (uint64_t)(((k >> 2) * kHalf + (k & 3) * 32) >> 4);
          umma_f16(t_dp + dp_buf(q) * 128, dr1 + off, tile + off, id_s, k != 0);
        }
        umma_commit(dp_full + dp_buf(q));
        if (!kKeyMajor) umma_commit(empty1 + st);         // V has no other reader
        return true;
      };
      // The first blocks of an item also wait for its resident tiles.  An item's last products of either kind free them.
      auto first_s = [&](uint32_t q) -> bool {
        if (!(wait(res_full, items & 1, 12) && issue_s(q, kThinItems && (w.flags & kThin) ? id_thin : id_s))) return false;
        if (w.n_it == 1) umma_commit(res_empty);
        return true;
      };
      auto first_dp = [&](uint32_t q) -> bool {
        if (!(wait(res_full + 1, items & 1, 12) && issue_dp(q, kThinItems && (w.flags & kThin) ? id_thin : id_s))) return false;
        if (w.n_it == 1) umma_commit(res_empty + 1);
        return true;
      };
      // acc += (P or dS in TMEM at `src`: a warp's columns packed from its first column) * streamed tile; the k-steps
      // of the first / second 16 columns of every warp
      auto issue_grad = [&](uint32_t acc, uint32_t src, uint64_t tile, int part, bool first) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          umma_f16_ts(acc, src + i * kBwdCols + part * 8, tile + (uint64_t)(((2 * i + part) * 2048) >> 4), id_g,
                      !(first && i == 0));
      };
      // Blocks follow one another across items: the next item's first S is issued where the next block's would be, and its
      // first dP behind this item's last product.
      ok = first_s(g) && first_dp(g);
      bool early = false;                                 // the next item's first S went before this item's last product
      while (ok && more) {
        const int n = w.n_it;
        const bool thin_item = kThinItems && (w.flags & kThin);
        for (int it = 0; it < n && ok; ++it, ++g) {
          const bool last = it + 1 == n;
          const uint32_t st0 = g % kRing0, st1 = g % kRing1;
          if (kKeyMajor) {
            // dV += P^T dO (contraction over the queries)
            if (!(ok = wait(p_ready, g & 1, 14))) break;
            issue_grad(t_acc0, tmem, ds1m + st1 * kStageOff, 0, it == 0);
            if (!(ok = wait(p_ready + 1, g & 1, 14))) break;
            issue_grad(t_acc0, tmem, ds1m + st1 * kStageOff, 1, false);
            umma_commit(empty1 + st1);
            if (last) umma_commit(acc_done);
          }
          if (!last) {
            if (!(ok = issue_s(g + 1, id_s))) break;
            if (it + 2 == n) umma_commit(res_empty);
            if (!kKeyMajor) {
              if (!(ok = issue_dp(g + 1, id_s))) break;
              if (it + 2 == n) umma_commit(res_empty + 1);
            }
          } else {
            more = next_item();                           // w is the next item's from here on
            mbar_arrive(clc_empty);
            // query-major, where the next item's tiles are there already: the element-wise warps get its scores behind their output
            early = !kKeyMajor && more && mbar_test(res_full, items & 1) && mbar_test(full0 + (g + 1) % kRing0, ((g + 1) / kRing0) & 1);
            if (early && !(ok = first_s(g + 1))) break;
          }
          if (!(ok = wait(ds_ready + (g & 1), (g >> 1) & 1, 14))) break;
          const uint32_t acc = kKeyMajor ? t_acc1 : t_acc0, ds = t_dp + dp_buf(g) * 128;
          if (it == 0 && thin_item) {
            umma_f16_ts(acc, ds, ds0m + st0 * kStageOff, id_g, false);
          } else {
            issue_grad(acc, ds, ds0m + st0 * kStageOff, 0, it == 0);   // dK += dS^T Q / dQ += dS K
            issue_grad(acc, ds, ds0m + st0 * kStageOff, 1, false);
          }
          umma_commit(empty0 + st0);
          if (last) umma_commit(acc_done + 1);
          if (last) {
            if (more && !early && !(ok = first_s(g + 1))) break;
            if (more && !(ok = first_dp(g + 1))) break;
          } else if (kKeyMajor) {
            if (!(ok = issue_dp(g + 1, id_s))) break;
            if (it + 2 == n) umma_commit(res_empty + 1);
          }
        }
      }
    }
  } else {
    const int q4 = warp & 3;
    const int part = (warp - 2) >> 2;                     // which kBwdCols of the 128 columns
    const int row = q4 * 32 + lane;                       // TMEM lane: key (key-major) or query
    const uint32_t lane_off = static_cast<uint32_t>(q4 * 32) << 16;
    const uint64_t sl2 = f32x2(a.scale * kLog2e, a.scale * kLog2e), sc2 = f32x2(a.scale, a.scale);
    bool more = true;
    float lse2 = 0.f, delta = 0.f;                        // query-major: this lane's statistics, asked for an item ahead
    auto ask = [&]() {
      if (!kKeyMajor) {
        const int64_t at = stat_at(a, w.b, w.h, w.blk) + row;
        lse2 = a.lse2[at];
        delta = a.delta[at];
      }
    };
    ask();
    while (more) {
      const int me = w.blk * kBlk + row;                  // query-major: this lane's query
      const int me0 = w.blk * kBlk + q4 * 32 + (lane >> 2);   // key-major: the first of this thread's keys
      const uint64_t my_lse2 = f32x2(lse2, lse2), my_delta = f32x2(delta, delta);
      Streamed<kKeyMajor> s(a, w);
      for (int it = 0; it < w.n_it; ++it, ++g, s.next(w)) {
        const uint32_t ts = tmem + lane_off + part * kBwdCols, tdp = ts + 128 + dp_buf(g) * 128;
        const int c0 = s.blk * kBlk + part * kBwdCols;   // first streamed index of this thread's columns
        const uint32_t st0 = g % kRing0;
        // key-major: lse2 / delta of this thread's columns
        const float* my_lse = sLse + st0 * kBlk + part * kBwdCols + (lane & 3) * 2;
        const float* my_dlt = sDelta + (g & 1) * kBlk + part * kBwdCols + (lane & 3) * 2;
        // only pairs on the diagonal or the window's edge, far ones with first tokens among the keys, and (key-major) those with queries
        // beyond the end, zeros whose score for an infinite key is NaN, pay for the mask
        const bool masked = kKeyMajor ? c0 < me0 + 24 || (c0 + kBwdCols - 1 - me0 >= a.window && me0 + 24 >= a.key_sinks) || c0 + kBwdCols > a.seq
                                      : c0 + kBwdCols - 1 > me || (me - c0 >= a.window && c0 + kBwdCols > a.sinks);
        // of a thin block only the first columns are there
        const bool mine = !kThinItems || it > 0 || part == 0 || !(w.flags & kThin);
        float e[kBwdCols];                                // P of this thread's columns
        // ---- phase 1: P = exp2(S * scale * log2(e) - lse2) ----
        // (key-major: lse2 comes with Q and delta with dO, whose barriers order them for this thread)
        if (!warp_wait(s_full, g & 1, 8 * tmo) || (kKeyMajor && !warp_wait(full0 + st0, (g / kRing0) & 1, 8 * tmo))) {
          if (lane == 0) report(a.status, kErrWindow + 15, it, 0);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        if (!mine) {
          if (lane == 0) mbar_arrive(s_free);
        } else {
          uint32_t rs[kBwdCols];
          if (kKeyMajor) {
            tmem_ld_16x32_frag(ts, rs);
            tmem_ld_16x32_frag(ts + (16u << 16), rs + 16);
          } else {
            tmem_ld_32x32(ts, rs);
          }
          tmem_ld_wait();
          if (!kKeyMajor) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free);           // the next block's S may be computed
          }
          uint64_t st[4] = {my_lse2, my_lse2, my_lse2, my_lse2};
          if (kKeyMajor) {
#pragma unroll
            for (int n = 0; n < 4; ++n) st[n] = *reinterpret_cast<const uint64_t*>(my_lse + n * 8);
          }
          // What is seen, as bits.  key-major: of query - key = base + 8 (n - r) + (0 or 1), in rising order; what is seen lies between
          // 0 and the window, for first tokens of any number above.
          uint32_t seen[4] = {};
          if (masked && kKeyMajor) {
            const int base = c0 + (lane & 3) * 2 - me0;
            const uint32_t from = ~low_bits(below(-base)), upto = low_bits(below(a.window - base));
#pragma unroll
            for (int r = 0; r < 4; ++r) seen[r] = me0 + r * 8 < a.key_sinks ? from : from & upto;
            if (c0 + kBwdCols > a.seq) {
#pragma unroll
              for (int r = 0; r < 4; ++r) seen[r] &= low_bits(below(a.seq - c0 - (lane & 3) * 2 - r * 8));
            }
          }
          if (masked && !kKeyMajor)
            seen[0] = low_bits(me - c0 + 1) & (~low_bits(me - c0 + 1 - a.window) | low_bits(a.sinks - c0));
          // key-major: columns of a fragment are in groups n of 8, elements 4 n + {0, 1} of this thread's first row of a
          // lane half, + {2, 3} of its second; by halves of 16 columns, so that P^T can be handed over in two parts
#pragma unroll
          for (int hp = 0; hp < 2; ++hp) {
#pragma unroll
            for (int i = 0; i < kBwdCols / 2; i += 2) {
              const int k = kKeyMajor ? (i >> 3) * 16 + hp * 8 + (i & 7) : hp * 16 + i;
              const uint64_t x = fma2(f32x2(__uint_as_float(rs[k]), __uint_as_float(rs[k + 1])), sl2, st[(k >> 2) & 3]);
              if (kKeyMajor && i % 8 < kBwdPoly) {
                exp2_poly(x, e[k], e[k + 1]);
              } else {
                split(x, e[k], e[k + 1]);
                e[k] = fast_exp2(e[k]);
                e[k + 1] = fast_exp2(e[k + 1]);
              }
            }
            if (masked) {
#pragma unroll
              for (int i = 0; i < kBwdCols / 2; ++i) {
                const int k = kKeyMajor ? (i >> 3) * 16 + hp * 8 + (i & 7) : hp * 16 + i;
                // key-major: row r of four (keys + 8 r), column group n of four (queries + 8 n): distance t = n - r
                const int r = (k >> 4) * 2 + (k >> 1 & 1), bit = kKeyMajor ? ((k >> 2 & 3) - r + 3) * 2 + (k & 1) : k;
                if (!(seen[kKeyMajor ? r : 0] >> bit & 1)) e[k] = 0.f;
              }
            }
            if (kKeyMajor) {
              // P^T over this warp's own S^T columns, packed from the first: the products that read the first 16
              // run under the exponentials of the second
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t pk[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pk[i] = pack_bf16(e[h * 16 + hp * 8 + 2 * i], e[h * 16 + hp * 8 + 2 * i + 1]);
                tmem_st_16x16_frag(ts + hp * 8 + ((h * 16u) << 16), pk);
              }
              tmem_st_wait();
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(p_ready + hp);
            }
          }
        }
        // ---- phase 2: dS = P * (dP * scale - delta * scale) ----
        if (!warp_wait(dp_full + dp_buf(g), dp_phase(g), 8 * tmo) ||
            (kKeyMajor && !warp_wait(full1 + (g & 1), (g >> 1) & 1, 8 * tmo))) {
          if (lane == 0) report(a.status, kErrWindow + 16, it, 0);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        if (!mine) {
          if (lane == 0) mbar_arrive(ds_ready + (g & 1));
        } else {
          uint32_t rp[kBwdCols], dk[16];
          uint64_t st[4] = {my_delta, my_delta, my_delta, my_delta};
          if (kKeyMajor) {
            tmem_ld_16x32_frag(tdp, rp);
            tmem_ld_16x32_frag(tdp + (16u << 16), rp + 16);
#pragma unroll
            for (int n = 0; n < 4; ++n) st[n] = *reinterpret_cast<const uint64_t*>(my_dlt + n * 8);
          } else {
            tmem_ld_32x32(tdp, rp);
          }
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < kBwdCols; k += 2) {
            float g0, g1;
            split(mul2(f32x2(e[k], e[k + 1]),
                       fma2(f32x2(__uint_as_float(rp[k]), __uint_as_float(rp[k + 1])), sc2, st[(k >> 2) & 3])), g0, g1);
            dk[k >> 1] = pack_bf16(g0, g1);
          }
          // dS over this thread's own dP columns
          if (kKeyMajor) {
            tmem_st_16x32_frag(tdp, dk);
            tmem_st_16x32_frag(tdp + (16u << 16), dk + 8);
          } else {
            tmem_st_32x16(tdp, dk);
          }
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(ds_ready + (g & 1));
        }
      }
      if (!ok) break;
      // Accumulators -> bf16 rows of dqkv: a warp's 32 rows x kBwdCols columns leave through shared memory as a TMA store
      // (with plain stores the warps stall for 4000 cycles when all SMs write their items at the same time).
      const int col = (kKeyMajor ? col_k(a, w.h) : col_q(a, w.kv, w.h)) + part * kBwdCols, orow = w.blk * kBlk + q4 * 32, ob = w.b;
      // what far queries add to a first token's gradients: this lane's row
      const float* far = kKeyMajor && a.far != nullptr && orow + lane < a.sinks
                             ? a.far + ((int64_t)w.b * a.kv + w.h) * kRowsPart + (orow + lane) * kD + part * kBwdCols : nullptr;
      const uint32_t phase = items & 1;
      // where the item's last dO or V was; dK: where its last Q was
      const uint32_t out_st = (g - 1) & 1, out_st0 = (g - 1) % kRing0;
      uint8_t* const stages[2] = {sS1 + out_st * kTile + (warp - 2) * kBwdStage,
                                  (kKeyMajor ? sS0 + out_st0 * kTile : sS1 + out_st * kTile) + (warp - 2) * kBwdStage};
      more = next_item();                        // w is the next item's from here on
      if (more) ask();
      __syncwarp();                              // every lane has read the slot: the one after may be asked for now
      if (lane == 0) mbar_arrive(clc_empty);
#pragma unroll 1
      for (int which = kKeyMajor ? 0 : 1; which < 2; ++which) {
        if (!warp_wait(acc_done + which, phase, 8 * tmo)) {
          if (lane == 0) report(a.status, kErrWindow + 17, which, 0);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        // key-major: acc0 = dV, acc1 = dK;  query-major: acc0 = dQ
        uint32_t r[kBwdCols];
        tmem_ld_32x32((kKeyMajor && which ? t_acc1 : t_acc0) + lane_off + part * kBwdCols, r);
        uint8_t* stage = stages[which];
        tmem_ld_wait();
        if (kKeyMajor && far != nullptr) {
          const float4* add = reinterpret_cast<const float4*>(far + which * kThinKeys * kD);
#pragma unroll
          for (int i = 0; i < kBwdCols / 4; ++i) {
            const float4 v = add[i];
            r[4 * i] = __float_as_uint(__uint_as_float(r[4 * i]) + v.x);
            r[4 * i + 1] = __float_as_uint(__uint_as_float(r[4 * i + 1]) + v.y);
            r[4 * i + 2] = __float_as_uint(__uint_as_float(r[4 * i + 2]) + v.z);
            r[4 * i + 3] = __float_as_uint(__uint_as_float(r[4 * i + 3]) + v.w);
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 v;
          v.x = pack_bf16(__uint_as_float(r[q * 8 + 0]), __uint_as_float(r[q * 8 + 1]));
          v.y = pack_bf16(__uint_as_float(r[q * 8 + 2]), __uint_as_float(r[q * 8 + 3]));
          v.z = pack_bf16(__uint_as_float(r[q * 8 + 4]), __uint_as_float(r[q * 8 + 5]));
          v.w = pack_bf16(__uint_as_float(r[q * 8 + 6]), __uint_as_float(r[q * 8 + 7]));
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) = v;   // 64-byte swizzle
        }
        warp_store_box(&tm_dqkv, stage, col + (kKeyMajor && which == 0 ? kD : 0), orow, ob, a.seq);
      }
      if (!ok) break;
      if (lane == 0) {                           // the stages may take tiles again
        if (kKeyMajor) {
          bulk_wait_read<1>();
          mbar_arrive(out_read + out_st);
          bulk_wait_read<0>();
          mbar_arrive(out_read0 + out_st0);
        } else {
          bulk_wait_read<0>();
          mbar_arrive(out_read + out_st);
        }
      }
      tc_fence_before_sync();                    // the accumulators are read before the next P / dS is announced
      __syncwarp();
    }
  }
  tc_fence_before_sync();
  __syncwarp();
  const bool all = __syncthreads_and(ok) != 0;
  tc_fence_after_sync();
  if (threadIdx.x == 0 && all)
    for (int i = 2; i < 35; ++i)
      if (i != 30) mbar_inval(bars + i);
  return all;
}

// A grid of key-major items, of query-major ones, or of both, all key-major items first; a CTA of both kinds changes when cluster
// launch control gives it an item of the other one, in that order at most once; nothing depends on that.
template <bool kKey, bool kQuery>
__global__ void __launch_bounds__(kBwdThreads, 1)
window_bwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_do,
                  const __grid_constant__ CUtensorMap tm_dqkv, const __grid_constant__ CUtensorMap tm_thin,
                  const __grid_constant__ WinBwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  // the base is 1024-byte aligned in practice; there is no room for the full slack of an arbitrary one
  if (smem - smem_raw > kBwdAlignSlack) {
    grid_wait();
    if (threadIdx.x == 0) report(a.status, kErrWindow + 10, 0, 0);
    return;
  }
  uint8_t* clc_resp = smem + kBwdBars;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kBwdBars + 30 * 8);
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_qkv);
    tma_prefetch_desc(&tm_do);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_wait();

  if (kKey && kQuery) {
    uint32_t item = blockIdx.x, y, z;
    bool more = true;
    while (more) {
      const bool ok = item < a.items ? window_bwd_run<true, false>(tm_qkv, tm_do, tm_dqkv, tm_thin, a, smem, tmem, item)
                                     : window_bwd_run<false, false>(tm_qkv, tm_do, tm_dqkv, tm_thin, a, smem, tmem, item);
      more = ok && clc_read(clc_resp, item, y, z);
      fence_proxy_async_smem();             // this read before the next response overwrites it
    }
  } else {
    window_bwd_run<kKey, !kKey>(tm_qkv, tm_do, tm_dqkv, tm_thin, a, smem, tmem, blockIdx.x);
  }
  if (warp >= 2 && warp < 2 + kBwdWarps && lane == 0) bulk_wait_all<0>();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// The shared-memory attribute is per device: set it once on every device that launches.
cudaError_t configure_device() {
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && configured[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(window_fwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFwdSmem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(window_rows_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(window_rows_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem);
  if (e != cudaSuccess) return e;
  for (auto kernel : {window_bwd_kernel<true, true>, window_bwd_kernel<true, false>, window_bwd_kernel<false, true>}) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBwdSmem);
    if (e != cudaSuccess) return e;
  }
  if (dev >= 0 && dev < 64) configured[dev] = true;
  return cudaSuccess;
}

int sm_count() {
  static int count[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (count[dev] == 0 && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return count[dev];
}

// Rows of items dealt together: the largest divisor of their number that is at most 32.
int deal(int n) {
  int g = 1;
  for (int d = 1; d <= 32; ++d)
    if (n % d == 0) g = d;
  return g;
}

bool off(const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0; }
int blocks_of(int seq) { return (seq + kBlk - 1) / kBlk; }
cudaError_t check(const WindowShape& s) {
  if (s.batch <= 0 || s.seq <= 0 || s.kv <= 0 || s.group <= 0 || s.window < 0 || s.sinks < 0) return cudaErrorInvalidValue;
  const int64_t rows = (int64_t)s.batch * s.kv * s.group, width = (int64_t)s.kv * (s.group + 2) * kD;
  if (rows > 65535 || blocks_of(s.seq) > 65535 || width > 1 << 24) return cudaErrorInvalidValue;
  return rows * blocks_of(s.seq) > 1 << 26 ? cudaErrorInvalidValue : cudaSuccess;
}

}  // namespace

cudaError_t window_attention_fwd(const void* qkv, void* out, float* lse, const WindowShape& s, uint32_t* status, cudaStream_t stream) {
  cudaError_t e = check(s);
  if (e != cudaSuccess) return e;
  if (off(qkv, 16) || off(out, 16)) return cudaErrorInvalidValue;
  e = configure_device();
  if (e != cudaSuccess) return e;
  const int heads = s.kv * s.group, nblk = blocks_of(s.seq);
  CUtensorMap tq, to, tt;
  const uint64_t width = (uint64_t)s.kv * (s.group + 2) * kD;
  if (make_tensor_map_seq(&tq, qkv, width, s.seq, s.batch, 64, kBlk) != 0) return cudaErrorInvalidValue;
  const bool thin = s.sinks > 0 && s.sinks <= kThinKeys && s.seq > kBlk;
  if (!thin) tt = tq;
  else if (make_tensor_map_seq(&tt, qkv, width, s.seq, s.batch, 64, kThinKeys) != 0) return cudaErrorInvalidValue;
  if (make_tensor_map_seq(&to, out, (uint64_t)heads * kD, s.seq, s.batch, 64, 32) != 0) return cudaErrorInvalidValue;
  WinArgs a{};
  a.batch = s.batch; a.seq = s.seq; a.kv = s.kv; a.group = s.group; a.heads = heads;
  a.window = s.window == 0 || s.window > s.seq ? s.seq : s.window;
  a.sinks = s.sinks < s.seq ? s.sinks : s.seq;
  a.thin = thin ? 1 : 0;
  a.scale = s.scale;
  a.lse = lse;
  a.status = status;
  a.timeout_ns = 2000000000ull;
  // With no more tiles than SMs a tile per CTA leaves none idle; beyond that pairs share K and V and overlap.
  a.tiles_per_item = (int64_t)s.batch * heads * nblk <= sm_count() ? 1 : 2;
  const int grp = deal(s.batch * heads);
  const dim3 grid(grp, (nblk + a.tiles_per_item - 1) / a.tiles_per_item, s.batch * heads / grp);
  return launch_dependent(window_fwd_kernel, grid, kFwdThreads, kFwdSmem, stream, tq, to, tt, a);
}

namespace {
// Few first tokens beyond a window: CTAs of window_rows_kernel per key head (0: the general way).  One wave of two CTAs an SM, each with
// a tile or more for every warp (the whole backward of 4 x 2048, 32 heads by CTAs an SM: 2 293 us, 3 299, 4 296, 7 300; 2 x 5003, 16 heads on 4: 267, 273,
// 275, 286).
int thin_chunks(const WindowShape& s) {
  if (s.batch <= 0 || s.kv <= 0) return 0;           // (such a launch is refused)
  if (s.sinks == 0 || s.sinks > kThinKeys || s.window == 0 || s.window >= s.seq) return 0;
  const int units = s.batch * s.kv, tiles = s.group * blocks_of(s.seq) * (kBlk / 16);
  int n = 148 * 2 / units;
  n = n < tiles / kRowsWarps ? n : tiles / kRowsWarps;
  return n < 1 ? 1 : n;
}
}  // namespace

int64_t window_attention_scratch(const WindowShape& s) {
  return 2 * (int64_t)s.batch * s.kv * s.group * blocks_of(s.seq) * kBlk + (int64_t)s.batch * s.kv * (thin_chunks(s) + 1) * kRowsPart;
}

cudaError_t window_attention_bwd(const void* qkv, const void* out, const void* dout, const float* lse, void* dqkv, float* scratch,
                                 const WindowShape& s, uint32_t* status, cudaStream_t stream) {
  cudaError_t e = check(s);
  if (e != cudaSuccess) return e;
  if (off(qkv, 16) || off(out, 16) || off(dout, 16) || off(dqkv, 16) || off(scratch, 16)) return cudaErrorInvalidValue;
  e = configure_device();
  if (e != cudaSuccess) return e;
  const int heads = s.kv * s.group, nblk = blocks_of(s.seq);
  const uint64_t width = (uint64_t)s.kv * (s.group + 2) * kD;
  CUtensorMap tq, td, tg, tt;
  if (make_tensor_map_seq(&tq, qkv, width, s.seq, s.batch, 64, kBlk) != 0) return cudaErrorInvalidValue;
  if (make_tensor_map_seq(&td, dout, (uint64_t)heads * kD, s.seq, s.batch, 64, kBlk) != 0) return cudaErrorInvalidValue;
  if (make_tensor_map_seq(&tg, dqkv, width, s.seq, s.batch, kBwdCols, 32) != 0) return cudaErrorInvalidValue;
  tt = tq;
  if (thin_chunks(s) > 0 && make_tensor_map_seq(&tt, qkv, width, s.seq, s.batch, 64, kThinKeys) != 0) return cudaErrorInvalidValue;
  WinBwdArgs g{};
  float* delta = scratch + (int64_t)s.batch * heads * nblk * kBlk;
  const int chunks = thin_chunks(s);
  if (chunks > 0) {
    const int tiles = s.group * nblk * (kBlk / 16);
    RowsArgs r{};
    r.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv);
    r.out = reinterpret_cast<const __nv_bfloat16*>(out);
    r.dout = reinterpret_cast<const __nv_bfloat16*>(dout);
    r.lse = lse;
    r.lse2 = scratch;
    r.delta = delta;
    r.parts = delta + (int64_t)s.batch * heads * nblk * kBlk;
    r.seq = s.seq; r.padded = nblk * kBlk; r.kv = s.kv; r.group = s.group; r.window = s.window; r.sinks = s.sinks < s.seq ? s.sinks : s.seq;
    r.per = (tiles + chunks - 1) / chunks;
    r.scale = s.scale;
    auto kernel = r.sinks > 8 ? window_rows_kernel<2> : window_rows_kernel<1>;
    e = launch_dependent(kernel, dim3((unsigned)chunks, (unsigned)(s.batch * s.kv)), kRowsWarps * 32, kRowsSmem, stream, r);
    if (e != cudaSuccess) return e;
    g.far = r.parts;
    if (chunks > 1) {
      float* sums = r.parts + (int64_t)s.batch * s.kv * chunks * kRowsPart;
      e = launch_dependent(window_parts_kernel, dim3(kRowsPart / 128, (unsigned)(s.batch * s.kv)), 128, 0, stream, r.parts, sums, chunks);
      if (e != cudaSuccess) return e;
      g.far = sums;
    }
  } else {
    const uint32_t groups = (uint32_t)((int64_t)s.batch * heads * nblk * (kBlk / kDeltaRows));
    e = launch_dependent(window_delta_kernel, (groups + 15) / 16, 256, 0, stream, reinterpret_cast<const uint4*>(out),
                         reinterpret_cast<const uint4*>(dout), delta, groups, (uint32_t)s.seq, (uint32_t)(nblk * kBlk), (uint32_t)heads,
                         lse, scratch, s.scale);
    if (e != cudaSuccess) return e;
  }
  g.lse2 = scratch;
  g.delta = delta;
  g.batch = s.batch; g.seq = s.seq; g.kv = s.kv; g.group = s.group; g.heads = heads;
  g.window = s.window == 0 || s.window > s.seq ? s.seq : s.window;
  g.sinks = s.sinks < s.seq ? s.sinks : s.seq;
  g.key_sinks = chunks > 0 ? 0 : g.sinks;
  g.scale = s.scale;
  g.status = status;
  g.timeout_ns = 2000000000ull;
  g.key_group = deal(s.batch * s.kv);
  g.query_group = deal(s.batch * heads);
  const uint32_t keys = (uint32_t)(s.batch * s.kv) * nblk, queries = (uint32_t)(s.batch * heads) * nblk;
  g.items = keys;
  // Both kinds in one launch up to six query-major items an SM, two launches beyond: in one, items of the second kind take the SMs that the
  // last of the first leave, but the kernel of both is slower by a few per cent.  Two / one, us: 1 x 2048, 12 heads, window 512 (192 items)
  // 43.1 / 36.4, 8 heads on 4 (256) 57.4 / 50.5; 2 x 3000, 16 on 8, window 500 (768) 127 / 119; 4 x 2048, 16 heads, window 512
  // (1024) 156 / 158; 2 x 5003, 16 on 4, window 1000 (1280) 271 / 276.
  if (queries <= 6u * sm_count())
    return launch_dependent(window_bwd_kernel<true, true>, keys + queries, kBwdThreads, kBwdSmem, stream, tq, td, tg, tt, g);
  e = launch_dependent(window_bwd_kernel<true, false>, keys, kBwdThreads, kBwdSmem, stream, tq, td, tg, tt, g);
  if (e != cudaSuccess) return e;
  g.items = 0;
  return launch_dependent(window_bwd_kernel<false, true>, queries, kBwdThreads, kBwdSmem, stream, tq, td, tg, tt, g);
}

}  // namespace msb
