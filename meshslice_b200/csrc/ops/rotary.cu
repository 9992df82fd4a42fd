// Rotary positions: each pair (a, b) of a query or key head becomes m (a cos t - b sin t, b cos t + a sin t), t = position *
// frequency.  The gradient is the same with -t.
#include "rotary.h"

#include <cuda_bf16.h>

#include "../common/pdl.cuh"
#include "../common/ptx.cuh"

namespace msb {

namespace {

constexpr int kThreads = 128;
constexpr int kUnit = 16;        // features per step of a thread: two 16-byte vectors, eight pairs
constexpr int kAhead = 4;        // steps whose loads are on their way together
constexpr int kMaxTokens = 32;   // per CTA

// n / d for 0 <= n < 2^31 by one multiplication: mul = ceil(2^(31 + bits) / d), 2^(bits - 1) < d <= 2^bits, whose excess over
// 2^(31 + bits) / d is below 1, so the quotient's is below n / 2^(31 + bits) <= 1 / d (Granlund and Montgomery).
struct Divisor {
  uint32_t d, mul, shift;
};
Divisor divisor(uint32_t d) {
  uint32_t bits = 0;
  while ((1ull << bits) < d) ++bits;
  Divisor v;
  v.d = d;
  v.shift = bits;
  v.mul = (uint32_t)(((1ull << (31 + bits)) + d - 1) / d);   // at most 2^31 (d = 1, powers of two) + 2^31
  return v;
}
__device__ __forceinline__ void divide(uint32_t n, const Divisor& d, uint32_t& q, uint32_t& r) {
  q = (uint32_t)(((uint64_t)n * d.mul) >> 31 >> d.shift);
  r = n - q * d.d;
}

struct Rows {
  RotaryArgs a;
  int per_cta;                 // tokens of a CTA
  int in_place;
  Divisor units, heads, group; // steps of a head; heads of a row that are visited; heads of a group in memory (or visited)
};

__device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
// Words of the two halves of four pairs (i, i + rot / 2): cs = cosine and sine of two pairs, t of either.
__device__ __forceinline__ void turn_halves(uint32_t& a, uint32_t& b, const float4& cs) {
  const float a0 = lo(a), a1 = hi(a), b0 = lo(b), b1 = hi(b);
  a = pack(a0 * cs.x - b0 * cs.y, a1 * cs.z - b1 * cs.w);
  b = pack(b0 * cs.x + a0 * cs.y, b1 * cs.z + a1 * cs.w);
}
__device__ __forceinline__ uint32_t turn_pair(uint32_t v, float c, float s) {
  return pack(lo(v) * c - hi(v) * s, hi(v) * c + lo(v) * s);
}

// A CTA takes a few tokens: first the cosines and sines of their positions, once for all heads, into shared memory, then the
// rows, 32 bytes a step.  The angle is counted in turns of 2^-64, where position * frequency wraps by itself and keeps 2^-32 of a
// turn at any position (in fp32 radians a position of 100000 is off by 0.004).
// Bound by HBM: it reads and writes the rows once (in place: the query and key heads).  8192 tokens of 96 heads of 128: 63.5 us, 6.3 TB/s
// (the tensor library's copy 63.7; with 256 threads a CTA 70.5, 512 72.4), in place 45; 16384 tokens of 24 heads 33.7 (copy 34.4).
template <bool kHalf>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const __grid_constant__ Rows w) {
  __shared__ float4 table[kMaxTokens * 32];         // [token][pair / 2 of a step][step]: tokens * rot_dim <= 128 * kMaxTokens
  const RotaryArgs& a = w.a;
  const int pairs = a.rot_dim >> 1, turned = a.rot_dim / kUnit;
  const int t0 = blockIdx.x * w.per_cta, tokens = min(w.per_cta, a.tokens - t0);
  grid_trigger();
  grid_wait();
  for (int p = threadIdx.x; p < tokens * pairs; p += kThreads) {
    const int t = p / pairs, i = p - t * pairs;
    const uint64_t pos = a.positions != nullptr ? (uint64_t)a.positions[t0 + t] : (uint64_t)((t0 + t) % a.seq);
    const int32_t part = (int32_t)((pos * a.turns[i]) >> 32);            // of a turn, in [-1/2, 1/2), times 2^32
    float s, c;
    sincospif((float)part * 4.656612873077393e-10f, &s, &c);             // 2^-31
    reinterpret_cast<float2*>(table + (t * 4 + ((i & 7) >> 1)) * turned + (i >> 3))[i & 1] =
        make_float2(c * a.factor, s * (a.factor * a.sign));
  }
  __syncthreads();
  const uint32_t steps = (uint32_t)tokens * w.heads.d * w.units.d;
  for (uint32_t i0 = threadIdx.x; i0 < steps; i0 += kThreads * kAhead) {
    uint4 u[kAhead], v[kAhead];
    uint4 *pu[kAhead], *pv[kAhead];
    int at[kAhead];                                                      // of the cosines, or -1: a copy
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t i = i0 + j * kThreads;
      if (i >= steps) break;
      uint32_t row, unit, t, head, pair, member;
      divide(i, w.units, row, unit);
      divide(row, w.heads, t, head);
      divide(head, w.group, pair, member);
      const int64_t first = (int64_t)(pair * (a.group + 2) + member) * a.head_dim;
      const bool turns = (int)unit < turned && (int)member <= a.group;
      const int o0 = kHalf && turns ? unit * 8 : unit * kUnit, o1 = kHalf && turns ? o0 + pairs : o0 + 8;
      const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x) + (t0 + t) * a.ldx + first;
      __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(a.y) + (t0 + t) * a.ldy + first;
      u[j] = ld_stream(reinterpret_cast<const uint4*>(x + o0));
      v[j] = ld_stream(reinterpret_cast<const uint4*>(x + o1));
      pu[j] = reinterpret_cast<uint4*>(y + o0);
      pv[j] = reinterpret_cast<uint4*>(y + o1);
      at[j] = turns ? t * 4 * turned + unit : -1;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * kThreads >= steps) break;
      if (at[j] >= 0) {
        float4 cs[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) cs[k] = table[at[j] + k * turned];
        if (kHalf) {
          turn_halves(u[j].x, v[j].x, cs[0]);
          turn_halves(u[j].y, v[j].y, cs[1]);
          turn_halves(u[j].z, v[j].z, cs[2]);
          turn_halves(u[j].w, v[j].w, cs[3]);
        } else {
          u[j] = make_uint4(turn_pair(u[j].x, cs[0].x, cs[0].y), turn_pair(u[j].y, cs[0].z, cs[0].w),
                            turn_pair(u[j].z, cs[1].x, cs[1].y), turn_pair(u[j].w, cs[1].z, cs[1].w));
          v[j] = make_uint4(turn_pair(v[j].x, cs[2].x, cs[2].y), turn_pair(v[j].y, cs[2].z, cs[2].w),
                            turn_pair(v[j].z, cs[3].x, cs[3].y), turn_pair(v[j].w, cs[3].z, cs[3].w));
        }
      }
      *pu[j] = u[j];
      *pv[j] = v[j];
    }
  }
}

}  // namespace

cudaError_t rotary(const RotaryArgs& a, cudaStream_t stream) {
  const auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (a.tokens <= 0 || a.seq <= 0 || a.kv <= 0 || a.group <= 0 || a.head_dim <= 0 || a.rot_dim <= 0) return cudaErrorInvalidValue;
  if (a.head_dim % kUnit || a.rot_dim % kUnit || a.rot_dim > a.head_dim || a.rot_dim > 256) return cudaErrorInvalidValue;
  const int64_t width = (int64_t)a.kv * (a.group + 2) * a.head_dim;
  if (off(a.x) || off(a.y) || a.ldx % 8 || a.ldy % 8 || a.ldx < width || a.ldy < width) return cudaErrorInvalidValue;
  if (width > 1 << 24) return cudaErrorInvalidValue;
  Rows w;
  w.a = a;
  w.in_place = a.x == a.y && a.ldx == a.ldy;
  // in place, only what turns is visited
  const int units = (w.in_place ? a.rot_dim : a.head_dim) / kUnit, members = w.in_place ? a.group + 1 : a.group + 2;
  w.units = divisor(units);
  w.heads = divisor(a.kv * members);
  w.group = divisor(members);
  // Enough tokens for eight steps a thread, so that the cosines of a CTA cost little beside them; fewer where that would leave
  // SMs without a CTA.
  const int row = units * a.kv * members;
  int per = 8 * kThreads / row;
  per = per < 1 ? 1 : per > kMaxTokens * 128 / a.rot_dim ? kMaxTokens * 128 / a.rot_dim : per;
  const int spread = (a.tokens + 148 * 4 - 1) / (148 * 4);
  w.per_cta = per < spread ? per : spread;
  if (w.per_cta > kMaxTokens) w.per_cta = kMaxTokens;
  const unsigned grid = (unsigned)((a.tokens + w.per_cta - 1) / w.per_cta);
  auto kernel = a.half ? rotary_kernel<true> : rotary_kernel<false>;
  return launch_dependent(kernel, grid, kThreads, 0, stream, w);
}

}  // namespace msb
