// Products with an epilogue of their own.  The roles are those of the plain GEMM of CTA pairs (sm100_gemm2.cu): a TMA producer warp
// per operand, one thread that issues every tcgen05.mma, four epilogue warps that drain one accumulator while the next tile is
// multiplied.  What differs is what the epilogue warps do with the fp32 sums, and where a tile's operands lie.
//
// Outputs leave in chunks of 32 rows x 32 columns: an epilogue warp stages up to 6 KiB of a chunk (three 16-bit boxes, or an fp32 and a
// 16-bit one) and has two such sets, so that the copy engine reads one while the other is written.  That takes one of the plain
// GEMM's pipeline stages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <string.h>

#include "../common/gate.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"
#include "pair.cuh"
#include "sm100_gemm.h"
#include "sm100_products.h"

namespace msb {

namespace {

constexpr uint32_t kAStageP = kBM * kBK * 2;
constexpr uint32_t b_stage_p(int bn) { return (bn / 2) * kBK * 2; }
constexpr uint32_t kBox16 = 32 * 64, kBox32 = 32 * 128;   // 32 x 32 of 16 and of 32 bits
constexpr uint32_t kSet = 3 * kBox16;                     // what a chunk stages at most
constexpr uint32_t kOutStageP = 4 * 2 * kSet;
constexpr int stages_p(int bn) { return bn == 256 ? 5 : 7; }
constexpr uint32_t smem_alloc_p(int bn) { return stages_p(bn) * (kAStageP + b_stage_p(bn)) + kOutStageP + 256 + 1024; }
constexpr int kThreadsP = 224;   // warps: A producer, MMA, 4x epilogue, B producer
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void report_p(const ProductArgs& a, uint32_t code, uint32_t d0, uint32_t d1) {
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

// The staging of an epilogue warp: two sets of boxes, written in turn.
struct ChunkStage {
  uint8_t* base;
  int turn;
  // The next set, free again: of the chunks sent so far only the last may still be read.
  __device__ __forceinline__ uint8_t* take(int lane) {
    if (lane == 0) bulk_wait_read<1>();
    __syncwarp();
    return base + (turn & 1) * kSet;
  }
  __device__ __forceinline__ void written() {
    fence_proxy_async_smem();
    __syncwarp();
    ++turn;
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

// What an epilogue warp knows of its tile.
struct TileAt {
  int item, m2, nb;        // item of the batch, 256-row block, column block
  int row0;                // first of this warp's 32 rows, in the item
  uint32_t taddr;          // its accumulator
  uint32_t drained;        // barrier to arrive at once it has been read
  int lane;
};
__device__ __forceinline__ void acc_drained(const TileAt& at) {
  tc_fence_before_sync();
  __syncwarp();
  if (at.lane == 0) mbar_arrive_cluster(at.drained);
}
__device__ __forceinline__ void send(const CUtensorMap* map, const uint8_t* box, int x, int y) { tma_store_box(map, box, x, y, false); }

// ---- kGated: columns [0, BN / 2) of the accumulator are the gate, the others the up projection of the same features ----
template <int BN>
__device__ __forceinline__ void epilogue_gated(const Product& p, const TileAt& at, ChunkStage& out) {
  constexpr int kChunks = BN / 2 / 32;
  const int chunks = (p.N + 31) / 32;
#pragma unroll 1
  for (int c = 0; c < kChunks; ++c) {
    float g[32], u[32];
    load_acc(at.taddr + c * 32, g);
    load_acc(at.taddr + BN / 2 + c * 32, u);
    if (c == kChunks - 1) acc_drained(at);
    const int col0 = at.nb * (BN / 2) + c * 32;
    if (at.row0 >= p.M || col0 >= p.N) continue;
    uint8_t* box = out.take(at.lane);
    uint32_t w[16];
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
    for (int i = 0; i < 16; ++i)
      w[i] = pk2(g[2 * i] * gate_sigmoid(g[2 * i], p.act) * u[2 * i], g[2 * i + 1] * gate_sigmoid(g[2 * i + 1], p.act) * u[2 * i + 1]);
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
}

// ---- kGatedGrad: the accumulator is dh; du = dh act(g), dg = dh u act'(g) ----
template <int BN>
__device__ __forceinline__ void epilogue_gated_grad(const Product& p, const TileAt& at, ChunkStage& out) {
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
  ask(at.nb * BN);
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    float v[32];
    load_acc(at.taddr + c * 32, v);
    if (c == BN / 32 - 1) acc_drained(at);
    const int col0 = at.nb * BN + c * 32;
    if (at.row0 >= p.M || col0 >= p.N) continue;
    const float fg = from_shared(e & 255u), fu = from_shared(e >> 8);
    uint32_t wg[16], wu[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 g = unh(xg[i]), u = unh(xu[i]);
      g.x *= fg; g.y *= fg; u.x *= fu; u.y *= fu;
      const float s0 = gate_sigmoid(g.x, p.act), s1 = gate_sigmoid(g.y, p.act);
      wu[i] = pk2(v[2 * i] * g.x * s0, v[2 * i + 1] * g.y * s1);
      wg[i] = pk2(v[2 * i] * u.x * gate_slope(g.x, s0, p.act), v[2 * i + 1] * u.y * gate_slope(g.y, s1, p.act));
    }
    if (c + 1 < BN / 32 && col0 + 32 < p.N) ask(col0 + 32);      // one chunk ahead
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
}

// ---- kPlain ----
template <int BN>
__device__ __forceinline__ void epilogue_plain(const Product& p, const TileAt& at, ChunkStage& out) {
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    float v[32];
    load_acc(at.taddr + c * 32, v);
    if (c == BN / 32 - 1) acc_drained(at);
    const int col0 = at.nb * BN + c * 32;
    if (at.row0 >= p.M || col0 >= p.N) continue;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pk2(v[2 * i], v[2 * i + 1]);
    uint8_t* box = out.take(at.lane);
    stage16(box, at.lane, w);
    out.written();
    if (at.lane == 0) {
      send(&p.o[0], box, col0, at.row0);
      bulk_commit();
    }
  }
}

// ---- kHead: a row's maximum over the tile's columns of the vocabulary, then its exponentials relative to that, which fp16 holds with
// 11 significant bits down to 2^-14 of the largest (in bf16 the second rounding, of the probabilities, would add to a first as large) ----
template <int BN>
__device__ __forceinline__ void epilogue_head(const Product& p, const TileAt& at, ChunkStage& out) {
  const int row = at.row0 + at.lane;
  const int first = at.nb * BN, valid = min(BN, p.vocab - first);      // may be negative: a tile of padding
  const bool live = at.row0 < p.M;
  int64_t y = -1;
  if (row < p.M) {
    const int64_t t = p.targets[row];
    y = t >= 0 && t < p.vocab ? t - first : -1;
  }
  float m = -CUDART_INF_F;
  if (live) {
#pragma unroll 1
    for (int c = 0; c < BN / 32; ++c) {
      if (c * 32 >= valid) break;
      float v[32];
      load_acc(at.taddr + c * 32, v);
      if (valid - c * 32 >= 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) m = fmaxf(m, v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) m = c * 32 + i < valid ? fmaxf(m, v[i]) : m;
      }
      if (y >= c * 32 && y < c * 32 + 32) {
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) z = y == c * 32 + i ? v[i] : z;
        p.label[row] = z;
      }
    }
  }
  const float ref = m == -CUDART_INF_F ? 0.f : m;               // nothing above -inf: exponentials of zero, not of NaN
  float s = 0.f;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col0 = first + c * 32;
    const bool wanted = live && (c * 32 < valid || (p.write && col0 < p.N));
    if (wanted) {
      float v[32];
      load_acc(at.taddr + c * 32, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = ex2((v[i] - ref) * kLog2e);   // the difference first: logits down to the type's lowest value
      if (valid - c * 32 < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c * 32 + i < valid ? v[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 32; i += 4) s += (v[i] + v[i + 1]) + (v[i + 2] + v[i + 3]);
      if (p.write) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pkh(v[2 * i], v[2 * i + 1]);
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
  acc_drained(at);
  if (row < p.M) p.stats[(int64_t)at.nb * p.M + row] = make_float2(m, s);
}

// ---- kGram: alpha acc + beta C in fp16; below the diagonal the tile is written a second time, mirrored ----
template <int BN>
__device__ __forceinline__ void epilogue_gram(const Product& p, const TileAt& at, ChunkStage& out) {
  const int64_t item0 = (int64_t)at.item * p.M;
  const int row = at.row0 + at.lane;
  const bool mirror = at.nb * BN + BN <= at.m2 * 2 * kBM;      // the tile has nothing on the diagonal
  __half* const whole = reinterpret_cast<__half*>(p.out) + item0 * p.M;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col0 = at.nb * BN + c * 32;
    const bool live = at.row0 < p.M && col0 < p.M;
    uint32_t x[16];
    if (live && p.c != nullptr) load_row16(reinterpret_cast<const __half*>(p.c) + (item0 + row) * p.M + col0, p.M - col0, x);
    float v[32];
    load_acc(at.taddr + c * 32, v);
    if (c == BN / 32 - 1) acc_drained(at);
    if (!live) continue;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 t = p.c != nullptr ? unh(x[i]) : make_float2(0.f, 0.f);
      w[i] = pkh(fmaf(p.beta, t.x, p.alpha * v[2 * i]), fmaf(p.beta, t.y, p.alpha * v[2 * i + 1]));
    }
    if (mirror) {
      unsigned short* at_t = reinterpret_cast<unsigned short*>(whole) + (int64_t)col0 * p.M + row;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        at_t[(int64_t)(2 * i) * p.M] = (unsigned short)(w[i] & 0xffffu);
        at_t[(int64_t)(2 * i + 1) * p.M] = (unsigned short)(w[i] >> 16);
      }
    }
    uint8_t* box = out.take(at.lane);
    stage16(box, at.lane, w);
    out.written();
    if (at.lane == 0) {
      send(&p.o[0], box, col0, (int)item0 + at.row0);
      bulk_commit();
    }
  }
}

// ---- kStep: alpha X + beta acc ----
template <int BN>
__device__ __forceinline__ void epilogue_step(const Product& p, const TileAt& at, ChunkStage& out) {
  const int64_t item0 = (int64_t)at.item * p.M;
  const int row = at.row0 + at.lane;
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    const int col0 = at.nb * BN + c * 32;
    const bool live = at.row0 < p.M && col0 < p.N;             // M and N are multiples of 64: whole chunks
    float4 x[8];
    if (live) {
      const float4* from = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.c) + (item0 + row) * p.N + col0);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = from[i];
    }
    float v[32];
    load_acc(at.taddr + c * 32, v);
    if (c == BN / 32 - 1) acc_drained(at);
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[4 * i] = fmaf(p.alpha, x[i].x, p.beta * v[4 * i]);
      v[4 * i + 1] = fmaf(p.alpha, x[i].y, p.beta * v[4 * i + 1]);
      v[4 * i + 2] = fmaf(p.alpha, x[i].z, p.beta * v[4 * i + 2]);
      v[4 * i + 3] = fmaf(p.alpha, x[i].w, p.beta * v[4 * i + 3]);
    }
    if (p.out == nullptr) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = pkh(v[2 * i] * p.scale, v[2 * i + 1] * p.scale);
      uint8_t* box = out.take(at.lane);
      stage32(box, at.lane, v);
      stage16(box + kBox32, at.lane, w);
      out.written();
      if (at.lane == 0) {
        send(&p.o[0], box, col0, (int)item0 + at.row0);
        send(&p.o[1], box + kBox32, col0, (int)item0 + at.row0);
        bulk_commit();
      }
      continue;
    }
    if (row >= p.rows) continue;
    const int64_t at0 = at.item * p.out_item + row * p.out_row + col0 * p.out_col;
    const int n = min(32, p.cols - col0);
    if (p.out_fp32) {
      float* o = reinterpret_cast<float*>(p.out) + at0;
      if (n == 32 && p.out_col == 1 && aligned16(o)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<float4*>(o)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < n) o[i * p.out_col] = v[i];
      }
    } else {
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.out) + at0;
      if (n == 32 && p.out_col == 1 && aligned16(o)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<uint4*>(o)[i] = make_uint4(pk2(v[8 * i], v[8 * i + 1]), pk2(v[8 * i + 2], v[8 * i + 3]),
                                                      pk2(v[8 * i + 4], v[8 * i + 5]), pk2(v[8 * i + 6], v[8 * i + 7]));
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < n) o[i * p.out_col] = __float2bfloat16_rn(v[i]);
      }
    }
  }
}

template <int Kind, int BN>
__device__ __forceinline__ void epilogue(const Product& p, const TileAt& at, ChunkStage& out) {
  if constexpr (Kind == kGated) epilogue_gated<BN>(p, at, out);
  if constexpr (Kind == kGatedGrad) epilogue_gated_grad<BN>(p, at, out);
  if constexpr (Kind == kPlain) epilogue_plain<BN>(p, at, out);
  if constexpr (Kind == kHead) epilogue_head<BN>(p, at, out);
  if constexpr (Kind == kGram) epilogue_gram<BN>(p, at, out);
  if constexpr (Kind == kStep) epilogue_step<BN>(p, at, out);
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
  constexpr bool kF16 = K0 == kGram || K0 == kStep;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr uint32_t kSmemB = kStagesP * kAStageP;
  constexpr uint32_t kSmemOut = kSmemB + kStagesP * kBStageP;
  uint8_t* sA = smem;
  uint8_t* sB = smem + kSmemB;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kSmemOut + kOutStageP);    // [kStagesP], used in the leader
  uint64_t* empty_bar = full_bar + kStagesP;     // [kStagesP], one set per CTA
  uint64_t* tfull_bar = empty_bar + kStagesP;    // [2], one set per CTA
  uint64_t* tempty_bar = tfull_bar + 2;          // [2], used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();      // 0: leader
  const uint64_t tmo = a.timeout_ns;
  const int num_tiles = a.tiles[2];
  const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
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
      mbar_init(tempty_bar + i, 8);  // a lane of each epilogue warp of both CTAs
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

  if (warp == 0 || warp == 6) {
    // ===================== TMA producers (both CTAs): warp 0 loads A, warp 6 loads B ==========
    if (elect_one()) {
      const bool is_a = warp == 0;
      const uint32_t full0 = mapa_u32(smem_u32(full_bar), 0);     // the leader's barriers
      uint32_t stage = 0, phase = 0;
      bool ok = true, free = true;                                // `free`: the next stage was seen empty
      for (int t = cluster_id; t < num_tiles && ok; t += n_clusters) {
        int which, item, m2, nb;
        where(t, which, item, m2, nb);
        const Product& p = a.p[which];
        const bool gated = K0 == kGated;                          // gate and up come from two matrices, one for each CTA
        const bool mn_major = (is_a ? p.a_mn_major : p.b_mn_major) != 0, map3d = (is_a ? p.a_map3d : p.b_map3d) != 0;
        const int first = item * (is_a ? p.a_item : p.b_item);    // of the item's rows in the map
        const int row = (is_a ? (2 * m2 + (int)rank) * kBM : gated ? nb * (BN / 2) : nb * BN + (int)rank * (BN / 2)) + (mn_major ? 0 : first);
        const int k_first = mn_major ? first : 0;
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
      for (int t = cluster_id; t < num_tiles && ok; t += n_clusters, ++it) {
        const uint32_t acc = it & 1, acc_phase = (it >> 1) & 1;
        if (!mbar_wait(tempty_bar + acc, acc_phase ^ 1, 6 * tmo)) {
          report_p(a, kTimeoutTmemEmpty, t, acc);
          ok = false;
          break;
        }
        const uint32_t tmem_d = tmem_base + acc * BN;
        const Product& p = a.p[K1 == kNone ? 0 : t >= a.tiles[1] ? 2 : t >= a.tiles[0] ? 1 : 0];
        const int kblocks = p.kblocks[0] + p.kblocks[1];
        const bool a_mn = p.a_mn_major != 0, b_mn = p.b_mn_major != 0;
        const uint32_t idesc = make_idesc_bf16(2 * kBM, BN, a_mn, b_mn) & (kF16 ? ~((1u << 7) | (1u << 10)) : ~0u);
        const uint64_t da0 = make_smem_desc(smem_u32(sA), a_mn ? kBK * 128 : 16, 1024);
        const uint64_t db0 = make_smem_desc(smem_u32(sB), b_mn ? kBK * 128 : 16, 1024);
        const uint32_t da_hi = (uint32_t)(da0 >> 32), db_hi = (uint32_t)(db0 >> 32);
        const uint32_t a_kstep = (a_mn ? 16 * 128 : 32) >> 4;
        const uint32_t b_kstep = (b_mn ? 16 * 128 : 32) >> 4;
        for (int kb = 0; kb < kblocks; ++kb) {
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
            umma_f16_pair(tmem_d, desc_at(da_lo + k * a_kstep, da_hi), desc_at(db_lo + k * b_kstep, db_hi), idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit_both(eb);                 // the stage is free in both CTAs
        }
        if (ok) umma_commit_both(smem_u32(tfull_bar + acc));
      }
    }
  } else {
    // ===================== epilogue (both CTAs, own 128 rows) =====================
    const int q = warp & 3;
    ChunkStage out{smem + kSmemOut + q * 2 * kSet, 0};
    int it = 0;
    for (int t = cluster_id; t < num_tiles; t += n_clusters, ++it) {
      int which, item, m2, nb;
      where(t, which, item, m2, nb);
      const uint32_t acc = it & 1, acc_phase = (it >> 1) & 1;
      int okw = 1;
      if (lane == 0) okw = mbar_wait(tfull_bar + acc, acc_phase, 7 * tmo) ? 1 : 0;
      okw = __shfl_sync(0xffffffffu, okw, 0);
      if (!okw) {
        if (lane == 0) report_p(a, kTimeoutTmemFull, t, acc);
        break;
      }
      mbar_wait(tfull_bar + acc, acc_phase, tmo);
      tc_fence_after_sync();
      const TileAt at{item, m2, nb, (2 * m2 + (int)rank) * kBM + q * 32, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN,
                      mapa_u32(smem_u32(tempty_bar + acc), 0), lane};
      if (K1 == kNone || which == 0) epilogue<K0, BN>(a.p[0], at, out);
      else epilogue<K1, BN>(a.p[which], at, out);
    }
    if (lane == 0) bulk_wait_all<0>();
  }

  // both CTAs are done with shared memory, barriers and TMEM of the pair
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

cudaError_t launch_sm100_products(ProductArgs& args, int k0, int k1, int problems, int tile_n, int sms, cudaStream_t stream) {
  int64_t tiles = 0;
  for (int i = 0; i < 3; ++i) {
    if (i < problems) tiles += product_tiles(args.p[i], i == 0 ? k0 : k1, tile_n);
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    args.tiles[i] = (int)tiles;
  }
  if (tiles == 0) return cudaSuccess;
  const int most = sms & ~1, grid = (int)(2 * tiles < most ? 2 * tiles : most);
#define MSB_PRODUCTS(A, B)                                                                           \
  if (k0 == A && k1 == B)                                                                            \
    return tile_n == 128 ? launch_as<A, B, 128>(args, grid, stream) : launch_as<A, B, 256>(args, grid, stream);
  MSB_PRODUCTS(kGated, kNone)
  MSB_PRODUCTS(kGatedGrad, kNone)
  MSB_PRODUCTS(kPlain, kNone)
  MSB_PRODUCTS(kHead, kNone)
  MSB_PRODUCTS(kGram, kNone)
  MSB_PRODUCTS(kStep, kNone)
#undef MSB_PRODUCTS
  return cudaErrorInvalidValue;
}

}  // namespace msb
