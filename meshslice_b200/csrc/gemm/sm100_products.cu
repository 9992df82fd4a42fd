// Products with an epilogue of their own.  The roles are those of the plain GEMM of CTA pairs (sm100_gemm2.cu): a TMA producer warp
// per operand, one thread that issues every tcgen05.mma, epilogue warps that drain one accumulator while the next tile is
// multiplied.  What differs is what the epilogue warps do with the fp32 sums, and where a tile's operands lie.
//
// There are eight epilogue warps, two for every 32 rows, which take half of a tile's columns each: the arithmetic of a chunk (32 rows x
// 32 columns) is a chain of latencies, and one warp a scheduler leaves it idle.  Outputs leave chunk by chunk as TMA stores from 6 or 8 KiB
// of staging a warp: as many sets of boxes as fit, written in turn (three 16-bit boxes are one set).  The staging
// takes one of the plain GEMM's pipeline stages.  What an epilogue reads of memory it asks for one chunk ahead, for the first chunk
// before the accumulator is complete.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <string.h>

#include "../common/gate.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "../common/store_row.cuh"
#include "pair.cuh"
#include "sm100_gemm.h"
#include "sm100_products.h"

namespace msb {

namespace {

constexpr uint32_t kAStageP = kBM * kBK * 2;
constexpr uint32_t b_stage_p(int bn) { return (bn / 2) * kBK * 2; }
constexpr uint32_t kBox16 = 32 * 64, kBox32 = 32 * 128;   // 32 x 32 of 16 and of 32 bits
constexpr int kEpiWarps = 8;
constexpr uint32_t staging(int bn) { return (bn == 256 ? 4 : 3) * kBox16; }       // of an epilogue warp
constexpr int stages_p(int bn) { return bn == 256 ? 5 : 7; }
constexpr uint32_t smem_alloc_p(int bn) { return stages_p(bn) * (kAStageP + b_stage_p(bn)) + kEpiWarps * staging(bn) + 256 + 1024; }
constexpr int kThreadsP = 32 * (3 + kEpiWarps);   // warps: A producer, MMA, epilogue, B producer
constexpr float kLog2e = 1.4426950408889634f;

template <class Args>
__device__ __forceinline__ void report_p(const Args& a, uint32_t code, uint32_t d0, uint32_t d1) {
  if (atomicCAS(a.status, 0u, code) == 0u) {
    a.status[1] = blockIdx.x;
    a.status[2] = d0;
    a.status[3] = d1;
  }
}

__device__ __forceinline__ uint32_t pkh(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unh(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The staging of an epilogue warp: sets of `kBytes`, written in turn.
template <uint32_t kStaging, uint32_t kBytes>
struct ChunkStage {
  static constexpr int kSets = kStaging / kBytes;
  uint8_t* base;
  int turn;
  // The next set, free again: of the chunks sent so far only the last kSets - 1 may still be read.
  __device__ __forceinline__ uint8_t* take(int lane) {
    if (lane == 0) bulk_wait_read<kSets - 1>();
    __syncwarp();
    uint8_t* set = base + turn * kBytes;
    turn = turn + 1 == kSets ? 0 : turn + 1;
    return set;
  }
  __device__ __forceinline__ void written() {
    fence_proxy_async_smem();
    __syncwarp();
  }
};
// 32 x 32 of 16 bits with a 64-byte swizzle, of 32 bits with a 128-byte one; a lane holds a row.
__device__ __forceinline__ void stage16(uint8_t* box, int lane, const uint32_t (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<uint4*>(box + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
__device__ __forceinline__ void stage32(uint8_t* box, int lane, const float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<float4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
__device__ __forceinline__ void load_acc(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  __syncwarp();
  tmem_ld_32x32(taddr, r);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// 32 16-bit values of a row, which begin on a 16-byte boundary; those from `nvalid` on (a multiple of 8) are zeros.
__device__ __forceinline__ void load_row16(const void* p, int nvalid, uint32_t (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 x = 8 * q < nvalid ? ld_stream(reinterpret_cast<const uint4*>(p) + q) : make_uint4(0u, 0u, 0u, 0u);
    v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
  }
}

// What the gradient needs of gate and up is kept in 16 bits: 11 significant bits (fp16) beside 8 of bf16, in a range that 32 features
// of a row share: their largest finite magnitude becomes 2^14 .. 2^15.  Kept in bf16 the gradients would be 1.9 times as far off as
// rounding them once; like this 1.4 times, as the outputs of a product of rounded factors are.
__device__ __forceinline__ uint32_t shared_exponent(const float (&v)[32]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = fmaxf(m, fabsf(v[i]));
  if (m == CUDART_INF_F) {
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = fabsf(v[i]) < CUDART_INF_F ? fmaxf(m, fabsf(v[i])) : m;
  }
  return max(__float_as_uint(m) >> 23, 16u);
}
__device__ __forceinline__ float to_shared(uint32_t e) { return __uint_as_float((268u - e) << 23); }     // 2^(141 - e)
__device__ __forceinline__ float from_shared(uint32_t e) { return __uint_as_float((e - 14u) << 23); }    // 2^(e - 141)

// What an epilogue warp knows of its tile, and the half of the columns that is its own.
struct TileAt {
  int item, m2, nb;        // item of the batch, 256-row block, column block
  int row0;                // first of this warp's 32 rows, in the item
  int half;
  uint32_t taddr;          // the accumulator of its rows
  uint64_t* full;          // the accumulator is complete
  uint32_t phase;
  uint32_t drained;        // barrier to arrive at once this warp has read it
  uint64_t timeout_ns;
  int lane;
  uint64_t* written;        // of a chain: what the product before wrote may be read
  uint32_t written_phase;
  uint64_t* full0;          // barriers and accumulators of even parts, and the number of the first part
  uint32_t drained0, tmem0;
  int it;

  // The same with the accumulator of a later part of the contraction.
  template <int BN>
  __device__ __forceinline__ TileAt part(int k) const {
    TileAt t = *this;
    const uint32_t acc = (uint32_t)(it + k) & 1;
    t.taddr = tmem0 + acc * BN;
    t.full = full0 + acc;
    t.phase = (uint32_t)(it + k) >> 1 & 1;
    t.drained = drained0 + acc * 8;
    return t;
  }

  // Bounded; false: given up.
  __device__ __forceinline__ bool before() const {
    int ok = 1;
    if (lane == 0) ok = mbar_wait(written, written_phase, 7 * timeout_ns) ? 1 : 0;
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();                          // a shuffle orders no memory: the other lanes read behind the wait too
    return ok != 0;
  }
  // Bounded; false: given up.
  __device__ __forceinline__ bool wait() const {
    int ok = 1;
    if (lane == 0) ok = mbar_wait(full, phase, 7 * timeout_ns) ? 1 : 0;
    if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
    mbar_wait(full, phase, timeout_ns);
    tc_fence_after_sync();
    return true;
  }
  __device__ __forceinline__ void read() const {
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(drained);
  }
};
__device__ __forceinline__ void send(const CUtensorMap* map, const uint8_t* box, int x, int y) { tma_store_box(map, box, x, y, false); }

// ---- kGated: columns [0, BN / 2) of the accumulator are the gate, the others the up projection of the same features ----
template <int BN>
__device__ __forceinline__ bool epilogue_gated(const Product& p, const TileAt& at, ChunkStage<staging(BN), 3 * kBox16>& out) {
  constexpr int kChunks = BN / 2 / 32 / 2;                     // of this warp
  const int chunks = (p.N + 31) / 32;
  if (!at.wait()) return false;
#pragma unroll 1
  for (int c = at.half * kChunks; c < (at.half + 1) * kChunks; ++c) {
    float g[32], u[32];
    load_acc(at.taddr + c * 32, g);
    load_acc(at.taddr + BN / 2 + c * 32, u);
    if (c == (at.half + 1) * kChunks - 1) at.read();
    const int col0 = at.nb * (BN / 2) + c * 32;
    if (at.row0 >= p.M || col0 >= p.N) continue;
    uint32_t w[16];
    uint8_t* box = out.take(at.lane);
    if (p.keep) {
      const uint32_t eg = shared_exponent(g), eu = shared_exponent(u);
      const float fg = to_shared(eg), fu = to_shared(eu);
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pkh(g[2 * i] * fg, g[2 * i + 1] * fg);
      stage16(box + kBox16, at.lane, w);
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pkh(u[2 * i] * fu, u[2 * i + 1] * fu);
      stage16(box + 2 * kBox16, at.lane, w);
      if (at.row0 + at.lane < p.M) p.exps[(int64_t)(at.row0 + at.lane) * chunks + (col0 >> 5)] = (uint16_t)(eg | eu << 8);
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) u[i] *= g[i] * gate_sigmoid(g[i], p.act);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pk2(u[2 * i], u[2 * i + 1]);
    stage16(box, at.lane, w);
    out.written();
    if (at.lane == 0) {
      send(&p.o[0], box, col0, at.row0);
      if (p.keep) {
        send(&p.o[1], box + kBox16, col0, at.row0);
        send(&p.o[2], box + 2 * kBox16, col0, at.row0);
      }
      bulk_commit();
    }
  }
  return true;
}

// ---- kGatedGrad: the accumulator is dh; du = dh act(g), dg = dh u act'(g) ----
template <int BN>
__device__ __forceinline__ bool epilogue_gated_grad(const Product& p, const TileAt& at, ChunkStage<staging(BN), 2 * kBox16>& out) {
  constexpr int kChunks = BN / 32 / 2;
  const int chunks = (p.N + 31) / 32;
  const int64_t row = at.row0 + at.lane;
  const bool live = row < p.M;
  uint32_t xg[16], xu[16], e = 0;
  const auto ask = [&](int col0) {
    const int nvalid = live ? p.N - col0 : 0;
    load_row16(reinterpret_cast<const __half*>(p.g) + row * p.N + col0, nvalid, xg);
    load_row16(reinterpret_cast<const __half*>(p.u) + row * p.N + col0, nvalid, xu);
    e = nvalid > 0 ? p.exps[row * chunks + (col0 >> 5)] : 0x1010u;
  };
  const int first = at.nb * BN + at.half * (BN / 2);
  ask(first);
  if (!at.wait()) return false;
#pragma unroll 1
  for (int c = 0; c < kChunks; ++c) {
    float v[32];
    load_acc(at.taddr + at.half * (BN / 2) + c * 32, v);
    if (c == kChunks - 1) at.read();
    const int col0 = first + c * 32;
    if (at.row0 >= p.M || col0 >= p.N) continue;
    const float fg = from_shared(e & 255u), fu = from_shared(e >> 8);
    uint32_t wg[16], wu[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 g = unh(xg[i]), u = unh(xu[i]);
      g.x *= fg; g.y *= fg; u.x *= fu; u.y *= fu;
      const float s0 = gate_sigmoid(g.x, p.act), s1 = gate_sigmoid(g.y, p.act);
      wu[i] = pk2(v[2 * i] * (g.x * s0), v[2 * i + 1] * (g.y * s1));       // the bounded factor first, as in ops/gated.cu
      wg[i] = pk2(v[2 * i] * (u.x * gate_slope(g.x, s0, p.act)), v[2 * i + 1] * (u.y * gate_slope(g.y, s1, p.act)));
    }
    if (c + 1 < kChunks && col0 + 32 < p.N) ask(col0 + 32);
    uint8_t* box = out.take(at.lane);
    stage16(box, at.lane, wg);
    stage16(box + kBox16, at.lane, wu);
    out.written();
    if (at.lane == 0) {
      send(&p.o[0], box, col0, at.row0);
      send(&p.o[1], box + kBox16, col0, at.row0);
      bulk_commit();
    }
  }
  return true;
}

// ---- kPlain: alpha acc in bf16 or fp32, stored or added to what is there ----
template <int BN>
__device__ __forceinline__ bool epilogue_plain(const Product& p, const TileAt& at, ChunkStage<staging(BN), kBox32>& out) {
  constexpr int kChunks = BN / 32 / 2;
  const float alpha = p.alpha;
  const int64_t row = at.row0 + at.lane;
  const bool read = p.accumulate && !p.out_fp32;               // the copy engine adds fp32 values; bf16 ones are added before the rounding
  const int first = at.nb * BN + at.half * (BN / 2);
  uint32_t x[16];
  const auto ask = [&](int col0) {
    load_row16(reinterpret_cast<const __nv_bfloat16*>(p.c) + row * p.ldc + col0, read && row < p.M ? p.N - col0 : 0, x);
  };
  ask(first);
  if (!at.wait()) return false;
#pragma unroll 1
  for (int c = 0; c < kChunks; ++c) {
    float v[32];
    load_acc(at.taddr + at.half * (BN / 2) + c * 32, v);
    if (c == kChunks - 1) at.read();
    const int col0 = first + c * 32;
    if (at.row0 >= p.M || col0 >= p.N) continue;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= alpha;
    uint8_t* box = out.take(at.lane);
    if (p.out_fp32) {
      stage32(box, at.lane, v);
    } else {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = read ? pk2(v[2 * i] + blo(x[i]), v[2 * i + 1] + bhi(x[i])) : pk2(v[2 * i], v[2 * i + 1]);
      if (read && c + 1 < kChunks) ask(col0 + 32);
      stage16(box, at.lane, w);
    }
    out.written();
    if (at.lane == 0) {
      tma_store_box(&p.o[0], box, col0, at.item * p.out_item_rows + at.row0, p.out_fp32 && p.accumulate);
      bulk_commit();
    }
  }
  return true;
}

// ---- kHead: a row's maximum over this warp's columns of the vocabulary, then its exponentials relative to that, which fp16 holds with
// 11 significant bits down to 2^-14 of the largest (in bf16 the second rounding, of the probabilities, would add to a first as large).  The logits
// are in registers from the first look at the accumulator on.  Long contractions come in parts, which are added here: the tensor pipe cuts
// its sums off after every 16 products, towards zero, and over 4096 of them a loss was 1.5e-6 off, in the mean of its square ----
template <int BN>
__device__ __forceinline__ bool epilogue_head(const Product& p, const TileAt& at, ChunkStage<staging(BN), kBox16>& out) {
  constexpr int kChunks = BN / 32 / 2;
  const int row = at.row0 + at.lane, M = p.M;
  const int first = at.nb * BN + at.half * (BN / 2);
  const int valid = min(BN / 2, p.vocab - first);              // may be negative: padding alone
  const bool live = at.row0 < M, write = p.write != 0;
  int64_t y = -1;
  if (row < M) {
    const int64_t t = p.targets[row];
    y = t >= 0 && t < p.vocab ? t - first : -1;
  }
  float z[kChunks][32];
  for (int part = 0; part < p.parts; ++part) {
    const TileAt now = at.part<BN>(part);
    if (!now.wait()) return false;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (part == 0) {
        load_acc(now.taddr + at.half * (BN / 2) + c * 32, z[c]);
      } else {
        float v[32];
        load_acc(now.taddr + at.half * (BN / 2) + c * 32, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) z[c][i] += v[i];
      }
    }
    now.read();
  }
  if (!live || first >= p.N) return true;
  float m = -CUDART_INF_F;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (valid - c * 32 >= 32) {
      float a = fmaxf(z[c][0], z[c][1]), b = fmaxf(z[c][2], z[c][3]);
#pragma unroll
      for (int i = 4; i < 32; i += 4) {
        a = fmaxf(a, fmaxf(z[c][i], z[c][i + 1]));
        b = fmaxf(b, fmaxf(z[c][i + 2], z[c][i + 3]));
      }
      m = fmaxf(m, fmaxf(a, b));
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) m = c * 32 + i < valid ? fmaxf(m, z[c][i]) : m;
    }
    if (y >= c * 32 && y < c * 32 + 32) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) t = y == c * 32 + i ? z[c][i] : t;
      p.label[row] = t;
    }
  }
  const float ref = m == -CUDART_INF_F ? 0.f : m;               // nothing above -inf: exponentials of zero, not of NaN
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col0 = first + c * 32;
    if (c * 32 < valid || (write && col0 < p.N)) {
#pragma unroll
      for (int i = 0; i < 32; ++i) z[c][i] = ex2((z[c][i] - ref) * kLog2e);   // the difference first: logits down to the type's lowest value
      if (valid - c * 32 < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) z[c][i] = c * 32 + i < valid ? z[c][i] : 0.f;
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 32; ++i) sum[i & 3] += z[c][i];
      s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (write) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pkh(z[c][2 * i], z[c][2 * i + 1]);
        uint8_t* box = out.take(at.lane);
        stage16(box, at.lane, w);
        out.written();
        if (at.lane == 0) {
          send(&p.o[0], box, col0, at.row0);
          bulk_commit();
        }
      }
    }
  }
  if (row < M) p.stats[(int64_t)(2 * at.nb + at.half) * M + row] = make_float2(m, s);
  return true;
}

// A tile of 32 x 32 sums from lanes that hold rows to lanes that hold neighbouring columns: what is read and written of memory beside them then is
// in whole lines.  (As rows of 128 bytes a lane, the fp32 X of a step took 11 us a tile of 256 x 256; as boxes of the copy engine, with a fence of
// 550 cycles for each, 12.)
__device__ __forceinline__ void to_columns(uint8_t* tile, int lane, const float (&v)[32]) {
  __syncwarp();
  stage32(tile, lane, v);
  __syncwarp();
}
__device__ __forceinline__ float4 sums_of(const uint8_t* tile, int row, int unit) {
  return *reinterpret_cast<const float4*>(tile + row * 128 + ((unit ^ (row & 7)) << 4));
}

// ---- kGram: alpha acc + beta C in fp16; below the diagonal the tile is written a second time, mirrored ----
template <int BN>
__device__ __forceinline__ bool epilogue_gram(const Product& p, const TileAt& at, uint8_t* tile) {
  // fields of an argument that is chosen at run time would be read again after every store
  const int M = p.M;
  const float alpha = p.alpha, beta = p.beta;
  const __half* const C = reinterpret_cast<const __half*>(p.c);
  constexpr int kChunks = BN / 32 / 2;
  uint8_t* const mirrored = tile + kBox32;                     // the chunk as fp16
  const int64_t item0 = (int64_t)at.item * M;
  const int lr = at.lane >> 2, lu = at.lane & 3;               // rows lr, lr + 8 .., columns 8 lu ..
  const bool mirror = at.nb * BN + BN <= at.m2 * 2 * kBM;      // the tile has nothing on the diagonal
  __half* const whole = reinterpret_cast<__half*>(p.out) + item0 * M;
  const int first = at.nb * BN + at.half * (BN / 2);
  uint4 x[4];
  const auto ask = [&](int col0) {
    const bool there = C != nullptr && at.row0 < M && col0 < M;          // M is a multiple of 64: whole chunks
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = there ? ld_stream(reinterpret_cast<const uint4*>(C + (item0 + at.row0 + 8 * i + lr) * M + col0 + 8 * lu))
                   : make_uint4(0u, 0u, 0u, 0u);
  };
  if (C != nullptr && !at.before()) return false;
  ask(first);
  if (!at.wait()) return false;
#pragma unroll 1
  for (int c = 0; c < kChunks; ++c) {
    const int col0 = first + c * 32;
    float v[32];
    load_acc(at.taddr + at.half * (BN / 2) + c * 32, v);
    if (c == kChunks - 1) at.read();
    if (at.row0 >= M || col0 >= M) continue;
    to_columns(tile, at.lane, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + lr;
      const float4 s0 = sums_of(tile, r, 2 * lu), s1 = sums_of(tile, r, 2 * lu + 1);
      const float2 t0 = unh(x[i].x), t1 = unh(x[i].y), t2 = unh(x[i].z), t3 = unh(x[i].w);
      const uint4 o = make_uint4(pkh(fmaf(beta, t0.x, alpha * s0.x), fmaf(beta, t0.y, alpha * s0.y)),
                                 pkh(fmaf(beta, t1.x, alpha * s0.z), fmaf(beta, t1.y, alpha * s0.w)),
                                 pkh(fmaf(beta, t2.x, alpha * s1.x), fmaf(beta, t2.y, alpha * s1.y)),
                                 pkh(fmaf(beta, t3.x, alpha * s1.z), fmaf(beta, t3.y, alpha * s1.w)));
      *reinterpret_cast<uint4*>(whole + (int64_t)(at.row0 + r) * M + col0 + 8 * lu) = o;
      if (mirror) *reinterpret_cast<uint4*>(mirrored + r * 64 + ((lu ^ ((r >> 1) & 3)) << 4)) = o;
    }
    if (c + 1 < kChunks) ask(col0 + 32);
    if (mirror) {
      __syncwarp();
      unsigned short* to = reinterpret_cast<unsigned short*>(whole) + (int64_t)col0 * M + at.row0 + at.lane;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint4 o = *reinterpret_cast<const uint4*>(mirrored + at.lane * 64 + ((q ^ ((at.lane >> 1) & 3)) << 4));
        const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          to[(int64_t)(8 * q + 2 * k) * M] = (unsigned short)(w[k] & 0xffffu);
          to[(int64_t)(8 * q + 2 * k + 1) * M] = (unsigned short)(w[k] >> 16);
        }
      }
    }
  }
  return true;
}

// ---- kStep: alpha X + beta acc ----
template <int BN>
__device__ __forceinline__ bool epilogue_step(const Product& p, const TileAt& at, uint8_t* tile) {
  const int M = p.M, N = p.N;
  const float alpha = p.alpha, beta = p.beta, scale = p.scale;
  __half* const copy = reinterpret_cast<__half*>(p.copy);
  const bool last = p.out != nullptr;
  constexpr int kChunks = BN / 32 / 2;
  const int64_t row0 = (int64_t)at.item * M + at.row0;
  const int lr = at.lane >> 3, lu = at.lane & 7;               // rows lr, lr + 4 .., columns 4 lu ..
  const int first = at.nb * BN + at.half * (BN / 2);
  float* const whole = const_cast<float*>(reinterpret_cast<const float*>(p.c));
  float4 x[8];
  const auto ask = [&](int col0) {                               // M and N are multiples of 64: whole chunks
    if (at.row0 >= M || col0 >= N) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 u = ld_stream(reinterpret_cast<const uint4*>(whole + (row0 + 4 * i + lr) * N + col0 + 4 * lu));
      x[i] = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
    }
  };
  if (!at.before()) return false;
  ask(first);
  if (!at.wait()) return false;
#pragma unroll 1
  for (int c = 0; c < kChunks; ++c) {
    const int col0 = first + c * 32;
    float v[32];
    load_acc(at.taddr + at.half * (BN / 2) + c * 32, v);
    if (c == kChunks - 1) at.read();
    if (at.row0 >= M || col0 >= N) continue;
    to_columns(tile, at.lane, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + lr;
      const float4 t = sums_of(tile, r, lu);
      x[i] = make_float4(fmaf(alpha, x[i].x, beta * t.x), fmaf(alpha, x[i].y, beta * t.y), fmaf(alpha, x[i].z, beta * t.z),
                         fmaf(alpha, x[i].w, beta * t.w));
      if (!last) {
        const int64_t to = (row0 + r) * N + col0 + 4 * lu;
        *reinterpret_cast<float4*>(whole + to) = x[i];
        *reinterpret_cast<uint2*>(copy + to) =
            make_uint2(pkh(x[i].x * scale, x[i].y * scale), pkh(x[i].z * scale, x[i].w * scale));
      } else {
        *reinterpret_cast<float4*>(tile + r * 128 + ((lu ^ (r & 7)) << 4)) = x[i];
      }
    }
    if (c + 1 < kChunks) ask(col0 + 32);
    if (!last) continue;
    // the result, in any layout: back to lanes that hold rows
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 t = sums_of(tile, at.lane, q);
      v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
    }
    const int64_t row = at.row0 + at.lane;
    if (row < p.rows)
      store_row32(p.out, at.item * p.out_item + row * p.out_row + col0 * p.out_col, p.out_col, min(32, p.cols - col0), p.out_fp32 != 0, v);
  }
  return true;
}

// Bytes of a chunk's boxes.
constexpr uint32_t set_bytes(int kind) {
  return kind == kGated ? 3 * kBox16 : kind == kGatedGrad || kind == kPlain ? 2 * kBox16 : kBox16;
}
template <int Kind, int BN>
__device__ __forceinline__ bool epilogue(const Product& p, const TileAt& at, ChunkStage<staging(BN), set_bytes(Kind)>& out) {
  if constexpr (Kind == kGated) return epilogue_gated<BN>(p, at, out);
  if constexpr (Kind == kGatedGrad) return epilogue_gated_grad<BN>(p, at, out);
  if constexpr (Kind == kPlain) return epilogue_plain<BN>(p, at, out);
  if constexpr (Kind == kHead) return epilogue_head<BN>(p, at, out);
  return false;
}

// Blocks of columns of an item: tiles of kGated have gate and up of half as many features.
__host__ __device__ constexpr int columns_of(int kind, int bn) { return kind == kGated ? bn / 2 : bn; }
// Tiles of kGram: per 256-row block those whose columns begin before its last row.
__host__ __device__ __forceinline__ int gram_tiles(int blocks, int per) { return per * (blocks * (blocks + 1) / 2); }

// Tile t of a problem: item, 256-row block, column block.
template <int Kind, int BN>
__device__ __forceinline__ void place(const Product& p, int t, int& item, int& m2, int& nb) {
  const int tm = (p.M + 2 * kBM - 1) / (2 * kBM);
  if constexpr (Kind == kGram) {
    constexpr int per = 2 * kBM / BN;                            // column blocks per row block
    const int all = gram_tiles(tm, per);
    item = t / all;
    const int r = t - item * all;
    int i = (int)((sqrtf(8.f * (float)(r / per) + 1.f) - 1.f) * 0.5f);
    while (gram_tiles(i + 1, per) <= r) ++i;
    while (gram_tiles(i, per) > r) --i;
    m2 = i;
    nb = r - gram_tiles(i, per);
  } else {
    constexpr int cols = columns_of(Kind, BN);
    const int tn = (p.N + cols - 1) / cols;
    item = t / (tm * tn);
    tile2(t - item * tm * tn, tm, tn, p.group, p.along_n != 0, m2, nb);
  }
}

}  // namespace

template <int K0, int K1, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadsP, 1)
sm100_products_kernel(const __grid_constant__ ProductArgs a) {
  constexpr int kStagesP = stages_p(BN);
  constexpr uint32_t kBStageP = b_stage_p(BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr uint32_t kSmemB = kStagesP * kAStageP;
  constexpr uint32_t kSmemOut = kSmemB + kStagesP * kBStageP;
  uint8_t* sA = smem;
  uint8_t* sB = smem + kSmemB;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kSmemOut + kEpiWarps * staging(BN));    // [kStagesP], used in the leader
  uint64_t* empty_bar = full_bar + kStagesP;     // [kStagesP], one set per CTA
  uint64_t* tfull_bar = empty_bar + kStagesP;    // [2], one set per CTA
  uint64_t* tempty_bar = tfull_bar + 2;          // [2], used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();      // 0: leader
  const uint64_t tmo = a.timeout_ns;
  const TileWalk first_walk(blockIdx.x >> 1, gridDim.x >> 1, a.lead, a.tiles[2], a.rounds);
  // Tile t: its problem and its place in it.
  const auto where = [&](int t, int& which, int& item, int& m2, int& nb) {
    which = 0;
    if constexpr (K1 != kNone) which = t >= a.tiles[1] ? 2 : t >= a.tiles[0] ? 1 : 0;
    if (K1 == kNone || which == 0) place<K0, BN>(a.p[0], t, item, m2, nb);
    else place<K1, BN>(a.p[which], t - a.tiles[which - 1], item, m2, nb);
  };

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&a.p[0].a[0]);
    tma_prefetch_desc(&a.p[0].b[0]);
    for (int i = 0; i < kStagesP; ++i) {
      mbar_init(full_bar + i, 2);    // the leader's two producers announce their operand's bytes
      mbar_init(empty_bar + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull_bar + i, 1);
      mbar_init(tempty_bar + i, 2 * kEpiWarps);  // a lane of each epilogue warp of both CTAs
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2u * BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  cluster_sync_all();      // barriers of both CTAs are initialised before any remote arrival
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  grid_trigger();
  grid_wait();

  if (warp == 0 || warp == 2 + kEpiWarps) {
    // ===================== TMA producers (both CTAs): warp 0 loads A, the last one B ==========
    if (elect_one()) {
      const bool is_a = warp == 0;
      const uint32_t full0 = mapa_u32(smem_u32(full_bar), 0);     // the leader's barriers
      uint32_t stage = 0, phase = 0;
      bool ok = true, free = true;                                // `free`: the next stage was seen empty
      for (TileWalk walk = first_walk; walk.more() && ok; walk.next()) {
        const int t = walk.t;
        int which, item, m2, nb;
        where(t, which, item, m2, nb);
        const Product& p = a.p[which];
        const bool gated = K0 == kGated;                          // gate and up come from two matrices, one for each CTA
        const bool mn_major = (is_a ? p.a_mn_major : p.b_mn_major) != 0, map3d = (is_a ? p.a_map3d : p.b_map3d) != 0;
        const int first = item * (is_a ? p.a_item : p.b_item);    // of the item's rows in the map
        const int row = (is_a ? (2 * m2 + (int)rank) * kBM : gated ? nb * (BN / 2) : nb * BN + (int)rank * (BN / 2)) + (mn_major ? 0 : first);
        const int k_first = (mn_major ? first : 0) + item * p.k_item;
        const uint32_t bytes = is_a ? kAStageP : kBStageP;
        uint8_t* ring = is_a ? sA : sB;
        const int boxes = is_a ? kBM / 64 : BN / 128;
        const int k0_blocks = p.kblocks[0], kblocks = k0_blocks + p.kblocks[1];
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!free && !mbar_wait(empty_bar + stage, phase ^ 1, 5 * tmo)) {
            report_p(a, kTimeoutEmpty, t, kb);
            ok = false;
            break;
          }
          const bool second = kb >= k0_blocks;
          const CUtensorMap* map = is_a ? &p.a[second ? 1 : 0] : &p.b[gated ? rank : second ? 1 : 0];
          const int k0 = k_first + (second ? kb - k0_blocks : kb) * kBK;
          const uint32_t fb = full0 + stage * 8;
          if (rank == 0) mbar_expect_tx(full_bar + stage, 2 * bytes);
          uint8_t* dst = ring + stage * bytes;
          if (!mn_major) {
            tma_load_2d_pair(dst, map, fb, k0, row);
          } else if (map3d) {
            tma_load_3d_pair(dst, map, fb, 0, k0, row >> 6);
          } else {
            for (int j = 0; j < boxes; ++j) tma_load_2d_pair(dst + j * (kBK * 128), map, fb, row + j * 64, k0);
          }
          if (++stage == kStagesP) { stage = 0; phase ^= 1; }
          free = mbar_test(empty_bar + stage, phase ^ 1);
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (leader only) =====================
    if (rank == 0 && elect_one()) {
      uint32_t stage = 0, phase = 0;
      bool ok = true, full = false;                               // `full`: the next stage was seen complete
      int it = 0;
      for (TileWalk walk = first_walk; walk.more() && ok; walk.next()) {
        const int t = walk.t;
        const Product& p = a.p[K1 == kNone ? 0 : t >= a.tiles[1] ? 2 : t >= a.tiles[0] ? 1 : 0];
        const int kblocks = p.kblocks[0] + p.kblocks[1];
        const bool a_mn = p.a_mn_major != 0, b_mn = p.b_mn_major != 0;
        const uint32_t idesc = make_idesc_bf16(2 * kBM, BN, a_mn, b_mn);
        const uint64_t da0 = make_smem_desc(smem_u32(sA), a_mn ? kBK * 128 : 16, 1024);
        const uint64_t db0 = make_smem_desc(smem_u32(sB), b_mn ? kBK * 128 : 16, 1024);
        const uint32_t da_hi = (uint32_t)(da0 >> 32), db_hi = (uint32_t)(db0 >> 32);
        const uint32_t a_kstep = (a_mn ? 16 * 128 : 32) >> 4;
        const uint32_t b_kstep = (b_mn ? 16 * 128 : 32) >> 4;
        // the contraction in one accumulator, or (kHead) in parts of one each
        const int parts = K0 == kHead ? p.parts : 1, per = (kblocks + parts - 1) / parts;
        uint32_t acc = 0, tmem_d = 0;
        int left = 0;                           // k-blocks of the part
        for (int kb = 0; kb < kblocks; ++kb) {
          const bool first = left == 0;
          if (first) {
            left = min(per, kblocks - kb);
            acc = it & 1;
            tmem_d = tmem_base + acc * BN;
            if (!mbar_wait(tempty_bar + acc, (it >> 1 & 1) ^ 1, 6 * tmo)) {
              report_p(a, kTimeoutTmemEmpty, t, acc);
              ok = false;
              break;
            }
            ++it;
          }
          if (!full && !mbar_wait(full_bar + stage, phase, 4 * tmo)) {
            report_p(a, kTimeoutFull, t, kb);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t da_lo = (uint32_t)da0 + stage * (kAStageP >> 4);
          const uint32_t db_lo = (uint32_t)db0 + stage * (kBStageP >> 4);
          const uint32_t eb = smem_u32(empty_bar + stage);
          if (++stage == kStagesP) { stage = 0; phase ^= 1; }
          full = mbar_test(full_bar + stage, phase);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_f16_pair(tmem_d, desc_at(da_lo + k * a_kstep, da_hi), desc_at(db_lo + k * b_kstep, db_hi), idesc, !first || k != 0 ? 1u : 0u);
          umma_commit_both(eb);                 // the stage is free in both CTAs
          if (--left == 0) umma_commit_both(smem_u32(tfull_bar + acc));
        }
      }
    }
  } else {
    // ===================== epilogue (both CTAs, own 128 rows) =====================
    const int q = warp & 3, half = (warp - 2) >> 2;
    // a warp's chunks of either kind, in the same staging: all of one problem's are read before the next one's first is written
    uint8_t* const boxes = smem + kSmemOut + (warp - 2) * staging(BN);
    ChunkStage<staging(BN), set_bytes(K0)> out0{boxes, 0};
    ChunkStage<staging(BN), set_bytes(K1 == kNone ? K0 : K1)> out1{boxes, 0};
    int last = 0;
    int it = 0;
    for (TileWalk walk = first_walk; walk.more(); walk.next(), it += K0 == kHead ? a.p[0].parts : 1) {
      const int t = walk.t;
      int which, item, m2, nb;
      where(t, which, item, m2, nb);
      const uint32_t acc = it & 1, acc_phase = (it >> 1) & 1;
      const uint32_t tmem0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16), drained0 = mapa_u32(smem_u32(tempty_bar), 0);
      const TileAt at{item, m2, nb, (2 * m2 + (int)rank) * kBM + q * 32, half, tmem0 + acc * BN, tfull_bar + acc, acc_phase, drained0 + acc * 8, tmo, lane,
                      nullptr, 0u, tfull_bar, drained0, tmem0, it};
      bool done;
      if (K1 == kNone || which == 0) {
        done = epilogue<K0, BN>(a.p[0], at, out0);
      } else {
        if (last == 0) {
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
        done = epilogue<K1 == kNone ? K0 : K1, BN>(a.p[which], at, out1);
      }
      last = which;
      if (!done) {
        if (lane == 0) report_p(a, kTimeoutTmemFull, t, acc);
        break;
      }
    }
    if (lane == 0) bulk_wait_all<0>();
  }

  // both CTAs are done with shared memory, barriers and TMEM of the pair
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * BN) : "memory");
}

// The products of an orthogonal update, one after another for every matrix of a batch, in one launch.  Tiles are numbered step by step, product by
// product, matrix by matrix, and go round the CTA pairs; a tile's operands are the whole product before it of the same matrix, so its producers
// wait until all of its CTAs have counted themselves done (one counter a product and matrix, an arrival and a reader a CTA: with one for every
// warp 3 x 1000 x 520 took 208 us).  A pair comes to its tiles in their order and every tile waits for
// earlier ones alone, so that with all pairs on the GPU (a cooperative launch) the first unfinished tile can always go on.  What that saves over a
// launch a product: with several matrices no pair stands idle at the end of a product, where 8 x 1024 x 1024 (80, 80 and 128 tiles of 256 x 256 on
// 74 pairs) took two rounds each, and no launch between any two of them.
template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadsP, 1)
sm100_chain_kernel(const __grid_constant__ ChainArgs a) {
  constexpr int kStagesP = stages_p(BN);
  constexpr uint32_t kBStageP = b_stage_p(BN);
  constexpr int kAhead = 16;        // tiles that a producer may be ahead of the epilogue, and more: a stage holds a k-block, the accumulators two tiles
  static_assert(kStagesP + 3 < kAhead, "");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr uint32_t kSmemB = kStagesP * kAStageP;
  constexpr uint32_t kSmemOut = kSmemB + kStagesP * kBStageP;
  uint8_t* sA = smem;
  uint8_t* sB = smem + kSmemB;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kSmemOut + kEpiWarps * staging(BN));
  uint64_t* empty_bar = full_bar + kStagesP;
  uint64_t* tfull_bar = empty_bar + kStagesP;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* before_bar = tempty_bar + 2;         // [kAhead], one set per CTA: the product before that of a tile has been written
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(before_bar + kAhead);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();      // 0: leader
  const uint64_t tmo = a.timeout_ns;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const int of_gram = a.items * a.tiles[0], of_step = a.items * a.tiles[1], round = 2 * of_gram + of_step, all = a.steps * round;
  struct Place {
    const Product* p;
    int phase;               // 0: X X^T, 1: b A + c A^2, 2: a X + B X
    int t;                   // of the product
    int index;               // of the product, 3 a step
  };
  const auto where = [&](int t) {
    const int step = t / round, r = t - step * round;
    Place w;
    w.phase = r >= 2 * of_gram ? 2 : r >= of_gram ? 1 : 0;
    w.t = r - (w.phase == 2 ? 2 * of_gram : w.phase * of_gram);
    w.index = 3 * step + w.phase;
    w.p = w.phase == 0 ? &a.gram[step & 1] : w.phase == 1 ? &a.square : &a.step[step + 1 == a.steps ? 2 : step & 1];
    return w;
  };
  const auto counted = [&](int index, int item) { return a.counters + (int64_t)index * a.items + item; };
  // CTAs' parts of the product before, of one matrix.
  const auto target = [&](int phase) { return (uint32_t)(a.tiles[phase == 0 ? 1 : 0] * 2); };

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < kStagesP; ++i) {
      mbar_init(full_bar + i, 2);
      mbar_init(empty_bar + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull_bar + i, 1);
      mbar_init(tempty_bar + i, 2 * kEpiWarps);
    }
    for (int i = 0; i < kAhead; ++i) mbar_init(before_bar + i, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2u * BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0 || warp == 2 + kEpiWarps) {
    // ===================== TMA producers =====================
    if (elect_one()) {
      const bool is_a = warp == 0;
      const uint32_t full0 = mapa_u32(smem_u32(full_bar), 0);
      uint32_t stage = 0, phase = 0;
      bool ok = true, free = true;
      int it = 0;
      for (int t = cluster; t < all && ok; t += clusters, ++it) {
        const Place w = where(t);
        const Product& p = *w.p;
        int item, m2, nb;
        if (w.phase < 2) place<kGram, BN>(p, w.t, item, m2, nb);
        else place<kStep, BN>(p, w.t, item, m2, nb);
        // One thread of a CTA looks at the counter, the others at what it saw.
        uint64_t* const before = before_bar + it % kAhead;
        if (is_a && w.index > 0 && !wait_flag_geq_gpu(counted(w.index - 1, item), target(w.phase), 5 * tmo)) {
          report_p(a, kTimeoutChunk, t, w.index);
          break;
        }
        if (is_a) {
          mbar_arrive(before);
        } else if (!mbar_wait(before, it / kAhead & 1, 6 * tmo)) {
          report_p(a, kTimeoutChunk, t, w.index);
          break;
        }
        asm volatile("fence.proxy.async.global;" ::: "memory");              // what was written by stores is read by copies
        const bool mn_major = (is_a ? p.a_mn_major : p.b_mn_major) != 0;      // of a step's X: always the 3-D map
        const int first = item * (is_a ? p.a_item : p.b_item);
        const int row = (is_a ? (2 * m2 + (int)rank) * kBM : nb * BN + (int)rank * (BN / 2)) + (mn_major ? 0 : first);
        const int k_first = mn_major ? first : 0;
        const uint32_t bytes = is_a ? kAStageP : kBStageP;
        uint8_t* ring = is_a ? sA : sB;
        const CUtensorMap* map = is_a ? &p.a[0] : &p.b[0];
        const int kblocks = p.kblocks[0];
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!free && !mbar_wait(empty_bar + stage, phase ^ 1, 5 * tmo)) {
            report_p(a, kTimeoutEmpty, t, kb);
            ok = false;
            break;
          }
          const uint32_t fb = full0 + stage * 8;
          if (rank == 0) mbar_expect_tx(full_bar + stage, 2 * bytes);
          uint8_t* dst = ring + stage * bytes;
          if (!mn_major) tma_load_2d_pair(dst, map, fb, kb * kBK, row);
          else tma_load_3d_pair(dst, map, fb, 0, k_first + kb * kBK, row >> 6);
          if (++stage == kStagesP) { stage = 0; phase ^= 1; }
          free = mbar_test(empty_bar + stage, phase ^ 1);
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (leader only) =====================
    if (rank == 0 && elect_one()) {
      uint32_t stage = 0, phase = 0;
      bool ok = true, full = false;
      int it = 0;
      for (int t = cluster; t < all && ok; t += clusters, ++it) {
        const uint32_t acc = it & 1, acc_phase = (it >> 1) & 1;
        if (!mbar_wait(tempty_bar + acc, acc_phase ^ 1, 6 * tmo)) {
          report_p(a, kTimeoutTmemEmpty, t, acc);
          ok = false;
          break;
        }
        const uint32_t tmem_d = tmem_base + acc * BN;
        const Product& p = *where(t).p;
        const bool b_mn = p.b_mn_major != 0;
        const uint32_t idesc = make_idesc_bf16(2 * kBM, BN, 0, b_mn) & ~((1u << 7) | (1u << 10));      // fp16
        const uint64_t da0 = make_smem_desc(smem_u32(sA), 16, 1024);
        const uint64_t db0 = make_smem_desc(smem_u32(sB), b_mn ? kBK * 128 : 16, 1024);
        const uint32_t da_hi = (uint32_t)(da0 >> 32), db_hi = (uint32_t)(db0 >> 32);
        const uint32_t b_kstep = (b_mn ? 16 * 128 : 32) >> 4;
        const int kblocks = p.kblocks[0];
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!full && !mbar_wait(full_bar + stage, phase, 6 * tmo)) {
            report_p(a, kTimeoutFull, t, kb);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t da_lo = (uint32_t)da0 + stage * (kAStageP >> 4);
          const uint32_t db_lo = (uint32_t)db0 + stage * (kBStageP >> 4);
          const uint32_t eb = smem_u32(empty_bar + stage);
          if (++stage == kStagesP) { stage = 0; phase ^= 1; }
          full = mbar_test(full_bar + stage, phase);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_f16_pair(tmem_d, desc_at(da_lo + k * 2, da_hi), desc_at(db_lo + k * b_kstep, db_hi), idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit_both(eb);
        }
        if (ok) umma_commit_both(smem_u32(tfull_bar + acc));
      }
    }
  } else {
    // ===================== epilogue =====================
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* const boxes = smem + kSmemOut + (warp - 2) * staging(BN);
    bool ok = true;
    int it = 0;
    for (int t = cluster; t < all; t += clusters, ++it) {
      const Place w = where(t);
      int item, m2, nb;
      if (w.phase < 2) place<kGram, BN>(*w.p, w.t, item, m2, nb);
      else place<kStep, BN>(*w.p, w.t, item, m2, nb);
      const uint32_t acc = it & 1, acc_phase = (it >> 1) & 1;
      const TileAt at{item, m2, nb, (2 * m2 + (int)rank) * kBM + q * 32, half,
                      tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN, tfull_bar + acc, acc_phase,
                      mapa_u32(smem_u32(tempty_bar + acc), 0), tmo, lane,
                      before_bar + it % kAhead, (uint32_t)(it / kAhead & 1), tfull_bar, 0u, 0u, it};
      // a warp that has given up does no more work, and still comes to the barrier of the CTA's epilogue warps
      if (ok && !(w.phase < 2 ? epilogue_gram<BN>(*w.p, at, boxes) : epilogue_step<BN>(*w.p, at, boxes))) {
        if (lane == 0) report_p(a, kTimeoutTmemFull, t, acc);
        ok = false;
      }
      __syncwarp();
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");      // this CTA's part is written
      if (warp == 2 && lane == 0) red_add_release_gpu(counted(w.index, item), 1);
    }
  }

  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * BN) : "memory");
}

template <int K0, int K1, int BN>
static cudaError_t launch_as(const ProductArgs& args, int grid, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  constexpr int smem = (int)smem_alloc_p(BN);
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(sm100_products_kernel<K0, K1, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  return launch_dependent(sm100_products_kernel<K0, K1, BN>, grid, kThreadsP, smem, stream, args);
}

int product_operands(Product* p, int kind, int tile_n, const ProductOperand* a, const ProductOperand* b, int ranges, int64_t rows_a,
                     int64_t rows_b, const int64_t* K) {
  p->a_mn_major = a[0].mn_major;
  p->b_mn_major = b[0].mn_major;
  const int maps_b = kind == kGated ? 2 : ranges;
  const auto build = [&](CUtensorMap* maps, const ProductOperand* o, int n, bool contraction_of_each, int64_t rows, int box_rows, int* map3d) {
    int r = 0;
    *map3d = 0;
    if (!o[0].mn_major) {
      for (int i = 0; i < n && r == 0; ++i)
        r = make_tensor_map_2d(&maps[i], o[i].base, K[contraction_of_each ? i : 0], rows, o[i].ld * 2, kBK, box_rows);
      return r;
    }
    const auto k_rows = [&](int i) { return o[i].k_rows > 0 ? o[i].k_rows : K[contraction_of_each ? i : 0]; };
    bool three = true;
    for (int i = 0; i < n && three; ++i) three = make_tensor_map_mn3d(&maps[i], o[i].base, rows, k_rows(i), o[i].ld * 2, box_rows / 64) == 0;
    *map3d = three;
    if (three) return 0;
    for (int i = 0; i < n && r == 0; ++i) r = make_tensor_map_2d(&maps[i], o[i].base, rows, k_rows(i), o[i].ld * 2, 64, kBK);
    return r;
  };
  int r = build(p->a, a, ranges, true, rows_a, kBM, &p->a_map3d);
  if (r == 0) r = build(p->b, b, maps_b, kind != kGated, rows_b, tile_n / 2, &p->b_map3d);
  for (int i = 0; i < 2; ++i) p->kblocks[i] = i < ranges ? (int)((K[i] + kBK - 1) / kBK) : 0;
  return r;
}

int product_output(Product* p, int which, const void* base, int64_t cols, int64_t rows, int64_t ld, bool fp32) {
  return make_tensor_map_chunk(&p->o[which], base, cols, rows, ld, fp32);
}

int64_t product_tiles(const Product& p, int kind, int tile_n) {
  const int64_t tm = (p.M + 2 * kBM - 1) / (2 * kBM);
  if (kind == kGram) return (int64_t)p.items * gram_tiles((int)tm, 2 * kBM / tile_n);
  const int cols = columns_of(kind, tile_n);
  return p.items * tm * ((p.N + cols - 1) / cols);
}

cudaError_t launch_sm100_products(ProductArgs& args, int k0, int k1, int problems, int longer, int tile_n, int sms, cudaStream_t stream) {
  int64_t tiles = 0;
  for (int i = 0; i < 3; ++i) {
    if (i < problems) tiles += product_tiles(args.p[i], i == 0 ? k0 : k1, tile_n);
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    args.tiles[i] = (int)tiles;
  }
  if (tiles == 0) return cudaSuccess;
  const int most = sms & ~1, grid = (int)(2 * tiles < most ? 2 * tiles : most);
  const auto kblocks = [&](int i) {
    const Product& p = args.p[i];
    return walk_blocks((int64_t)p.kblocks[0] + p.kblocks[1], (i == 0 ? k0 : k1) == kPlain && p.accumulate && !p.out_fp32 ? kWalkAdded16 : kWalkStored);
  };
  args.lead = args.tiles[longer - 1];
  args.rounds = longer == problems ? 0 : (int)walk_rounds(args.lead, kblocks(0), args.tiles[2] - args.lead, kblocks(longer), grid / 2);
#define MSB_PRODUCTS(A, B)                                                                           \
  if (k0 == A && k1 == B)                                                                            \
    return tile_n == 128 ? launch_as<A, B, 128>(args, grid, stream) : launch_as<A, B, 256>(args, grid, stream);
  MSB_PRODUCTS(kGated, kNone)
  MSB_PRODUCTS(kGatedGrad, kPlain)
  MSB_PRODUCTS(kPlain, kGatedGrad)
  MSB_PRODUCTS(kPlain, kPlain)
  MSB_PRODUCTS(kHead, kNone)
#undef MSB_PRODUCTS
  return cudaErrorInvalidValue;
}


template <int BN>
static cudaError_t launch_chain_as(const ChainArgs& args, int64_t most_tiles, int sms, cudaStream_t stream) {
  static int resident[64] = {0};          // clusters that fit the GPU at a time, 0: not yet asked
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  constexpr int smem = (int)smem_alloc_p(BN);
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(kThreadsP);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  int clusters = dev < 64 ? resident[dev] : 0;
  if (clusters == 0) {
    e = cudaFuncSetAttribute(sm100_chain_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&clusters, sm100_chain_kernel<BN>, &cfg);
    if (e != cudaSuccess) return e;
    if (clusters < 1) return cudaErrorLaunchOutOfResources;
    if (dev < 64) resident[dev] = clusters;
  }
  int64_t n = clusters < sms / 2 ? clusters : sms / 2;
  n = most_tiles < n ? most_tiles : n;
  cfg.gridDim = dim3((unsigned)(2 * (n < 1 ? 1 : n)));
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sm100_chain_kernel<BN>, args);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e;
}

// Columns of a tile: with 256 fewer operand bytes and rounds, with 128 a shorter way from one product to the next.  Us with tiles of 128 and of 256
// columns, and how many of the latter a pair has in a step: 1024 x 1024 128 and 195 (0.5), 2048 x 2048 222 and 281 (1.8), 8 x 1024 x 1024 262 and
// 271 (3.9), 4 x 1024 x 4096 472 and 496 (4.5), 4096 x 4096 1318 and 1183 (7.1), 16 x 1024 x 1024 528 and 479 (7.8).
int chain_tile_n(int64_t m, int64_t n, int64_t items, int sms) {
  Product gram, step;
  gram.M = gram.N = step.M = (int)m;
  step.N = (int)n;
  gram.items = step.items = (int)items;
  return 2 * product_tiles(gram, kGram, 256) + product_tiles(step, kStep, 256) < 6 * (int64_t)(sms / 2) ? 128 : 256;
}

cudaError_t launch_sm100_chain(ChainArgs& args, int tile_n, int sms, cudaStream_t stream) {
  const int64_t gram = product_tiles(args.square, kGram, tile_n), step = product_tiles(args.step[0], kStep, tile_n);
  if (args.items < 1 || args.steps < 1 || (2 * gram + step) * args.steps > 0x3fffffff) return cudaErrorInvalidValue;
  args.tiles[0] = (int)(gram / args.items);
  args.tiles[1] = (int)(step / args.items);
  const int64_t most = gram > step ? gram : step;
  return tile_n == 128 ? launch_chain_as<128>(args, most, sms, stream) : launch_chain_as<256>(args, most, sms, stream);
}

}  // namespace msb
