// Distillation loss over rows of logits: softmax statistics, the teacher's few entries, the gradient.
#include "distill.h"

#include <cuda_bf16.h>
#include <float.h>

#include <type_traits>

#include "../common/f32x2.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"

namespace msb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kNegInf2 = 0xff80ff80u;       // two bf16 -inf
constexpr int kVec = 4;                          // vectors of a thread that are worked on together
constexpr int kRowBytes = 200 * 1024;            // most of a row that is kept

__device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint64_t unpack2(uint32_t v) { return f32x2(lo(v), hi(v)); }
__device__ __forceinline__ uint64_t both(float v) { return f32x2(v, v); }
__device__ __forceinline__ uint32_t pack(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
// Larger of two bf16, twice (a NaN only where both are NaN: the sums show the others).
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// 2^x in one instruction, results below 2^-126 zero: beside a largest term of 1 they are nothing.
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// The columns of vector v from `valid` on count as -inf.
__device__ __forceinline__ uint4 cut(uint4 u, int v, int valid) {
  if (v * 8 + 8 > valid) {
    uint32_t* w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (v * 8 + 2 * i >= valid) w[i] = kNegInf2;
      else if (v * 8 + 2 * i + 1 >= valid) w[i] = (w[i] & 0xffffu) | (kNegInf2 & 0xffff0000u);
    }
  }
  return u;
}

// Which exponentials a row needs: those of z / T, of z (one kind serves both where T = 1), both, or, where T = 2 or 4, those of z as the
// squares of those of z / T, or the squares of these: the special-function unit gives 16 a cycle and SM, so that four of them an element
// take 180 us for 4096 rows of 50257 (148 SMs), two 90 (temperature 3: 244 us, 2: 162).
enum Kind { kSoft = 1, kHard = 2, kTwo = 3, kSquare = 5, kFourth = 9 };
constexpr int powers(int K) { return K == kSquare ? 2 : K == kFourth ? 4 : 1; }

// 2^x exponents of z over a temperature: z c - m c with the product z c exact (one rounding, of the result) and m c rounded once for
// the whole row: `ref`, the same wherever m is.  Sums are relative to 2^ref; that ref is not quite m c cancels in every ratio, and the
// loss takes ref itself.
// That holds while ref is off by little (1 at kNear).  From there on, where masks of the type's lowest value or of -1e30 are, neighbours of
// bf16 are 2^16 or more apart in exponent: a term is 1, where z is m, or nothing.  Then c gives way to a power of two that brings m to
// 2^17: z and m scaled by it are exact, and neighbours still 2^9 apart.  Sums are relative to m itself.
constexpr float kNear = 16777216.f;
__device__ __forceinline__ float ref_of(float m, float c) { return __fmul_rn(m, c); }
__device__ __forceinline__ bool near(float ref) { return fabsf(ref) < kNear; }
struct Exponent {
  float c, ref;
};
__device__ __forceinline__ Exponent exponent_of(float m, float c) {
  Exponent e{c, ref_of(m, c)};
  if (!near(e.ref)) {
    e.c = __uint_as_float(min(271u - ((__float_as_uint(m) >> 23) & 255u), 254u) << 23);
    e.ref = m * e.c;
  }
  return e;
}
// What sums relative to m0 are times, relative to m1 > m0 (of the p-th powers of the terms).  From or to a far one nothing is left, also where
// both references are beyond fp32.
__device__ __forceinline__ float lowered(float m0, float m1, float c, float p = 1.f) {
  return exp2_ftz(fmaxf(p * ref_of(m0, c) - p * ref_of(m1, c), -200.f));
}

// A thread's running maximum m, and sums of exp(z) and exp(z / T) relative to it.  (Behind the exponentials scalar sums: packing their
// results takes moves.)
template <int K>
struct Sums {
  static constexpr bool soft_exp = K & kSoft, squares = powers(K) > 1;
  float m = -INFINITY, soft = 0.f, hard = 0.f;
  // Where T = 2 or 4 what the hard one is relative to is a power of what the soft one is.
  static __device__ __forceinline__ float soft_lowered(float m0, float m1, float c) { return lowered(m0, m1, c); }
  static __device__ __forceinline__ float hard_lowered(float m0, float m1, float c) {
    return squares ? lowered(m0, m1, c, powers(K)) : lowered(m0, m1, kLog2e);
  }
  // z less what the sums are relative to, of z / T and of z.
  __device__ __forceinline__ float soft_above(float z, float c) const {
    const float r = ref_of(m, c);
    return (near(r) ? fmaf(z, c, -r) : (z - m) * c) * kLn2;
  }
  __device__ __forceinline__ float hard_above(float z, float c) const {
    const float r = ref_of(m, squares ? c : kLog2e);
    return (near(r) ? fmaf(z, kLog2e, squares ? -powers(K) * r : -r) : (z - m) * kLog2e) * kLn2;
  }
  __device__ __forceinline__ void raise(float to, float c) {
    if (to > m) {
      soft *= soft_lowered(m, to, c);                     // (while m is -inf the sums are 0)
      hard *= hard_lowered(m, to, c);
      m = to;
    }
  }
  template <int N>
  __device__ __forceinline__ void add(const uint4 (&u)[N], float c) {
    uint32_t top = kNegInf2;
#pragma unroll
    for (int j = 0; j < N; ++j) top = max_bf16x2(max_bf16x2(max_bf16x2(top, u[j].x), max_bf16x2(u[j].y, u[j].z)), u[j].w);
    raise(fmaxf(lo(top), hi(top)), c);
    const float c0 = soft_exp ? c : kLog2e, r0 = ref_of(m, c0), r1 = ref_of(m, kLog2e);
    if (near(K == kTwo ? fmaxf(fabsf(r0), fabsf(r1)) : r0)) {
      const uint64_t cs = both(c0), rs = both(-r0), ch = both(kLog2e), rh = both(-r1);
      float ps[4] = {}, ph[4] = {};
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t z = unpack2(w[i]);
          const int at = (i & 1) * 2;
          float a, b;
          split(fma2(z, cs, rs), a, b);
          a = exp2_ftz(a);
          b = exp2_ftz(b);
          ps[at] += a;
          ps[at + 1] += b;
          if (squares) {
            if (K == kFourth) {
              a *= a;
              b *= b;
            }
            ph[at] = fmaf(a, a, ph[at]);
            ph[at + 1] = fmaf(b, b, ph[at + 1]);
          }
          if (K == kTwo) {
            split(fma2(z, ch, rh), a, b);
            ph[at] += exp2_ftz(a);
            ph[at + 1] += exp2_ftz(b);
          }
        }
      }
      const float p = (ps[0] + ps[1]) + (ps[2] + ps[3]);
      if (soft_exp) soft += p;
      else hard += p;
      if (K == kTwo || squares) hard += (ph[0] + ph[1]) + (ph[2] + ph[3]);
    } else {
      // far from zero, or everything seen is -inf: then nothing counts, except that a NaN has to show
      Exponent es = exponent_of(m, c0), eh = exponent_of(m, kLog2e);
      if (m == -INFINITY) es.ref = eh.ref = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = exp2_ftz(fmaf(lo(w[i]), es.c, -es.ref)), b = exp2_ftz(fmaf(hi(w[i]), es.c, -es.ref));
          if (soft_exp) soft += a + b;
          if (K == kTwo) hard += exp2_ftz(fmaf(lo(w[i]), eh.c, -eh.ref)) + exp2_ftz(fmaf(hi(w[i]), eh.c, -eh.ref));
          else if (!soft_exp || squares) hard += a + b;        // (powers of 1 and of nothing)
        }
      }
    }
  }
  // Those of the warp's lanes, left in red (3 * 32 floats) by each warp / those of `warps` warps, for every thread that comes to read.
  __device__ __forceinline__ void leave(float c, float* red) {
    const float mine = m;
    m = warp_max(m);
    // (a thread that has seen nothing but -inf has sums of 0, or NaN)
    const bool as_is = mine == m || mine == -INFINITY;
    soft = warp_sum(as_is ? soft : soft * soft_lowered(mine, m, c));
    hard = warp_sum(as_is ? hard : hard * hard_lowered(mine, m, c));
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) { red[w] = m; red[32 + w] = soft; red[64 + w] = hard; }
  }
  __device__ __forceinline__ void join(float c, const float* red, int warps) {
    const int l = threadIdx.x & 31;
    m = l < warps ? red[l] : -INFINITY;
    const float mine = m;
    m = warp_max(m);
    const bool as_is = mine == m || mine == -INFINITY;
    soft = warp_sum(l < warps ? red[32 + l] * (as_is ? 1.f : soft_lowered(mine, m, c)) : 0.f);
    hard = warp_sum(l < warps ? red[64 + l] * (as_is ? 1.f : hard_lowered(mine, m, c)) : 0.f);
    if (K == kSoft) hard = soft;             // T = 1, or the labels have no weight
    if (K == kHard) soft = hard;
  }
};

// The teacher's entries of a row in shared memory: the column of each (id in the vocabulary) and its probability.  Where a column has
// several entries the first has their sum, in their order, and the others column -1; no entry has -1 too.  Entry `top` is the label's
// column, with no probability of its own, unless an entry has it.
struct Entries {
  int* at;
  float* p;
};
__host__ __device__ constexpr int entry_bytes(int top) { return (top + 1 + 3) / 4 * 4 * 8; }
__device__ __forceinline__ Entries entries_at(void* at, int top) {
  Entries e;
  e.at = reinterpret_cast<int*>(at);
  e.p = reinterpret_cast<float*>(e.at + (top + 1 + 3) / 4 * 4);
  return e;
}
__device__ __forceinline__ float value_at(const DistillArgs& a, int64_t i) {
  return a.values_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.values)[i]) : reinterpret_cast<const float*>(a.values)[i];
}
// Whether a row has an entry of any weight, its label's column or -1, and sum p log p.
struct RowTarget {
  bool some;
  int label;
  float plogp;
};
// What a lane has of a row on its way from memory: entries lane + 32 j, all of them where the teacher kept no more than 32 kHeld.
constexpr int kHeld = 4;
struct Held {
  int64_t id[kHeld], label;
  float value[kHeld];
};
__device__ __forceinline__ Held hold(const DistillArgs& a, int row) {
  const int l = threadIdx.x & 31;
  const int64_t base = (int64_t)row * a.top;
  Held h;
  h.label = a.targets != nullptr ? a.targets[row] : -1;
  if (a.top <= 32 * kHeld) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int k = l + 32 * j;
      h.id[j] = k < a.top ? a.ids[base + k] : -1;
      h.value[j] = k < a.top ? value_at(a, base + k) : -INFINITY;
    }
  }
  return h;
}
// Entry k of a row whose ids are in raw: the first of its column?  Adds what later ones of the column have.
__device__ __forceinline__ bool first_of(const Entries& raw, int top, int k, float& p) {
  const int id = raw.at[k];
  if (id < 0) return false;
  const int4* quads = reinterpret_cast<const int4*>(raw.at);
  int same = 0;
#pragma unroll 4
  for (int q = 0; q < (top + 4) / 4; ++q) {
    const int4 o = quads[q];
    same += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
  }
  if (same == 1) return true;
  for (int j = 0; j <= top; ++j) {
    if (raw.at[j] != id || j == k) continue;
    if (j < k) return false;
    p += raw.p[j];
  }
  return true;
}
// By one warp: the entries of `row` (h: what is held of it), through `raw`.
__device__ __forceinline__ RowTarget read_entries(const DistillArgs& a, int row, const Held& h, const Entries& raw, const Entries& e) {
  const int l = threadIdx.x & 31;
  const float c = kLog2e / a.temperature;
  RowTarget t;
  t.label = h.label >= 0 && h.label < a.vocab ? (int)h.label : -1;
  t.plogp = 0.f;
  float mx = -INFINITY, sum = 0.f;
  if (a.top <= 32 * kHeld) {
    float p[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      p[j] = h.id[j] >= 0 && h.id[j] < a.vocab ? h.value[j] : -INFINITY;
      mx = p[j] > mx || p[j] != p[j] ? p[j] : mx;
    }
    mx = warp_max(mx);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      p[j] = p[j] == -INFINITY ? 0.f : exp2_ftz((p[j] - mx) * c);
      sum += p[j];
    }
    sum = warp_sum(sum);
    t.some = sum != 0.f;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int k = l + 32 * j;
      if (j * 32 > a.top) break;
      p[j] = t.some ? p[j] / sum : 0.f;
      if (p[j] != 0.f) t.plogp += p[j] * logf(p[j]);
      if (k < a.top) {
        raw.at[k] = h.id[j] >= 0 && h.id[j] < a.vocab ? (int)h.id[j] : -1;
        raw.p[k] = p[j];
      }
    }
  } else {
    const int64_t base = (int64_t)row * a.top;
    for (int k = l; k < a.top; k += 32) {
      const int64_t id = a.ids[base + k];
      const float v = value_at(a, base + k), x = id >= 0 && id < a.vocab ? v : -INFINITY;
      raw.at[k] = id >= 0 && id < a.vocab ? (int)id : -1;
      raw.p[k] = x;
      mx = x > mx || x != x ? x : mx;
    }
    mx = warp_max(mx);
    for (int k = l; k < a.top; k += 32) {
      const float x = raw.p[k] == -INFINITY ? 0.f : exp2_ftz((raw.p[k] - mx) * c);
      sum += x;
      raw.p[k] = x;
    }
    sum = warp_sum(sum);
    t.some = sum != 0.f;
    for (int k = l; k < a.top; k += 32) {
      const float p = t.some ? raw.p[k] / sum : 0.f;
      if (p != 0.f) t.plogp += p * logf(p);
      raw.p[k] = p;
    }
  }
  t.plogp = warp_sum(t.plogp);
  if (l < 4 && a.top + l < (a.top + 4) / 4 * 4) {       // the label, and what pads to whole vectors
    raw.at[a.top + l] = l == 0 ? t.label : -1;
    raw.p[a.top + l] = 0.f;
  }
  __syncwarp();
  for (int k = l; k <= a.top; k += 32) {
    float p = raw.p[k];
    e.at[k] = first_of(raw, a.top, k, p) ? raw.at[k] : -1;
    e.p[k] = p;
  }
  __syncwarp();
  return t;
}

// What the gradient of a row is made of: soft * 2^(z c - ref) + hard * 2^(z hard_c - hard_ref), less `drop` times an entry's
// probability and `label` at the label.  From sums relative to the same references.
struct Weights {
  float c, ref, hard_c, hard_ref, soft, hard, drop, label;
};
template <int K>
__device__ __forceinline__ Weights weights_of(const DistillArgs& a, float m, float soft, float hard, bool some, bool label) {
  Weights w;
  const Exponent es = exponent_of(m, K == kHard ? kLog2e : kLog2e / a.temperature), eh = exponent_of(m, kLog2e);
  w.c = es.c;
  w.ref = es.ref;
  w.hard_c = eh.c;
  w.hard_ref = eh.ref;
  w.drop = some ? (1.f - a.hard) * a.temperature * a.scale : 0.f;
  w.label = label ? a.hard * a.scale : 0.f;
  w.soft = w.drop / soft;
  w.hard = w.label / hard;
  if (K == kSoft) w.soft = a.temperature == 1.f ? w.soft + w.hard : w.soft;      // one kind of exponentials
  return w;
}
template <int K>
__device__ __forceinline__ float grad_of(float e, float hard, const Weights& w) {
  if (K == kSoft) return e * w.soft;
  if (K == kHard) return e * w.hard;
  if (K == kSquare) return e * fmaf(e, w.hard, w.soft);
  if (K == kFourth) return e * fmaf(e * e, e * w.hard, w.soft);
  return fmaf(e, w.soft, hard * w.hard);
}
template <int K>
__device__ __forceinline__ uint32_t grad_pair(uint32_t z, const Weights& w) {
  float a, b, x = 0.f, y = 0.f;
  split(fma2(unpack2(z), both(w.c), both(-w.ref)), a, b);
  if (K == kTwo) {
    split(fma2(unpack2(z), both(w.hard_c), both(-w.hard_ref)), x, y);
    x = exp2_ftz(x);
    y = exp2_ftz(y);
  }
  return pack(grad_of<K>(exp2_ftz(a), x, w), grad_of<K>(exp2_ftz(b), y, w));
}
template <int K>
__device__ __forceinline__ float grad_one(float z, const Weights& w) {
  return grad_of<K>(exp2_ftz(fmaf(z, w.c, -w.ref)), K == kTwo ? exp2_ftz(fmaf(z, w.hard_c, -w.hard_ref)) : 0.f, w);
}
template <int K>
__device__ __forceinline__ uint4 grad_whole(uint4 u, const Weights& w) {
  return make_uint4(grad_pair<K>(u.x, w), grad_pair<K>(u.y, w), grad_pair<K>(u.z, w), grad_pair<K>(u.w, w));
}
template <int K>
__device__ __forceinline__ uint4 grad_vector(uint4 u, int v, int valid, const Weights& w) {
  const uint4 g = grad_whole<K>(u, w);
  if (v * 8 + 8 <= valid) return g;
  uint32_t r[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = v * 8 + 2 * i >= valid ? 0u : v * 8 + 2 * i + 1 >= valid ? r[i] & 0xffffu : r[i];
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// What an entry takes off its column's gradient.
__device__ __forceinline__ float drop_of(const Weights& w, int at, float p, int label) {
  return w.drop * p + (at == label ? w.label : 0.f);
}
// A row's loss: cross = sum p (z / T - r) over its entries and their sum `total`, zy = z - h of its label, where r and h are what the
// sums are relative to.
__device__ __forceinline__ float loss_of(const DistillArgs& a, const RowTarget& t, float soft, float hard, float cross, float total, float zy) {
  float loss = 0.f;
  if (t.some && a.hard != 1.f) loss = (1.f - a.hard) * a.temperature * a.temperature * (t.plogp + total * logf(soft) - cross);
  if (t.label >= 0 && a.hard != 0.f) loss += a.hard * (logf(hard) - zy);
  return loss;
}

// The rows' barriers.
enum { kSums = 1, kTaken = 2, kWritten = 3 };
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// Whole rows: a row waits in shared memory between the sums and the gradient, so the logits are read once.  Persistent CTAs: a thread
// reads its own vectors in both passes, and as the gradient of one leaves, the same place takes that vector of the CTA's next row: loads
// run under both passes.  A warp more, the clerk, reads the next row's entries meanwhile, takes their logits out of the row before it is
// overwritten (kTaken), and writes their columns again once the row's gradient is written (kWritten).
// 4096 rows of 50257 at temperature 2: 165 us (5.1 TB/s; without arithmetic 142: the rows of an SM take turns between the passes).  One CTA a
// row that begins when the one before it ends 514; persistent with sixteen warps 216; entries held a row ahead and no work on vectors
// that are not there 183; by the widths below 172, with a row's copies in two groups instead of one for every four vectors 165.
// CTAs of an SM by width: a row that fills shared memory alone has sixteen warps, one of up to 8192 columns four; between, eight (4096 rows of
// 50257, two CTAs an SM: 16 warps 182 us, 12 175, 8 172, 4 200; 8192 of 8000: 8 warps 89 us, 4 78).
constexpr int row_ctas(int T) { return T == 512 ? 1 : T == 256 ? 3 : 7; }
template <int K, int T>
__global__ void __launch_bounds__(T + 32, row_ctas(T))
distill_row_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 ring[];
  __shared__ float red[2][96];
  __shared__ int has[2], labels[2];
  const int nvec = a.cols >> 3, valid = min(a.cols, a.vocab), nv = (valid + 7) >> 3;
  const float c = kLog2e / a.temperature;
  const __nv_bfloat16* kept = reinterpret_cast<const __nv_bfloat16*>(ring);
  auto out_row = [&](int row) { return reinterpret_cast<__nv_bfloat16*>(a.grad) + (int64_t)row * a.ldg; };
  grid_trigger();
  grid_wait();
  int parity = 0;
  if (threadIdx.x >= T) {
    const int l = threadIdx.x & 31;
    const Entries raw = entries_at(ring + nv, a.top);
    uint8_t* buffers = reinterpret_cast<uint8_t*>(ring + nv) + entry_bytes(a.top);
    auto rewrite = [&](int row, int buf) {
      bar_sync(kWritten, T + 32);
      const Entries e = entries_at(buffers + buf * entry_bytes(a.top), a.top);
      __nv_bfloat16* out = out_row(row);
      for (int k = l; k <= a.top; k += 32)
        if (e.at[k] >= 0) out[e.at[k]] = __float2bfloat16(e.p[k]);
    };
    Held held = hold(a, blockIdx.x);
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
      const Entries e = entries_at(buffers + parity * entry_bytes(a.top), a.top);
      const RowTarget t = read_entries(a, row, held, raw, e);
      if (row + (int)gridDim.x < a.rows) held = hold(a, row + gridDim.x);
      if (l == 0) {
        has[parity] = t.some;
        labels[parity] = t.label;
      }
      if (row != (int)blockIdx.x) rewrite(row - gridDim.x, parity ^ 1);
      bar_sync(kSums, T + 32);
      // the logits of the entries first: the other warps wait for it before the next row arrives
      for (int k = l; k <= a.top; k += 32) raw.p[k] = e.at[k] >= 0 ? __bfloat162float(kept[e.at[k]]) : 0.f;
      const float y = t.label >= 0 ? __bfloat162float(kept[t.label]) : 0.f;
      __syncwarp();
      bar_arrive(kTaken, T + 32);
      Sums<K> sum;
      sum.join(c, red[parity], T >> 5);
      const Weights w = weights_of<K>(a, sum.m, sum.soft, sum.hard, t.some, t.label >= 0);
      float cross = 0.f, total = 0.f;
      for (int k = l; k <= a.top; k += 32) {
        const int at = e.at[k];
        if (at < 0) continue;
        const float z = raw.p[k], p = e.p[k], drop = drop_of(w, at, p, t.label);
        if (p != 0.f) {
          cross += p * sum.soft_above(z, c);
          total += p;
        }
        if (drop == 0.f) e.at[k] = -1;                       // (its column is as the others)
        else e.p[k] = grad_one<K>(z, w) - drop;
      }
      cross = warp_sum(cross);
      total = warp_sum(total);
      if (l == 0) a.loss[row] = loss_of(a, t, sum.soft, sum.hard, cross, total, t.label >= 0 ? sum.hard_above(y, c) : 0.f);
    }
    const int rows = (a.rows - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    rewrite(blockIdx.x + (rows - 1) * gridDim.x, parity ^ 1);
    return;
  }
  // Whole groups of kVec vectors a thread need no tests; what is left is worked on by the warps that have something of it.  A row's copies
  // are two groups to wait for: the first `half` whole groups, the others.
  constexpr int kStep = kVec * T;
  const int whole = valid / (8 * kStep), half = whole >> 1, rest = threadIdx.x + whole * kStep;
  uint4* mine = ring + threadIdx.x;
  auto logits_row = [&](int row) {
    return reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.logits) + (int64_t)row * a.ld);
  };
  {
    const uint4* z = logits_row(blockIdx.x);
    for (int g = 0; g < whole; ++g) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) cp_async16(mine + g * kStep + j * T, z + threadIdx.x + g * kStep + j * T);
      if (g + 1 == half) cp_async_commit();
    }
    for (int v = rest; v < nv; v += T) cp_async16(ring + v, z + v);
    cp_async_commit();
  }
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
    Sums<K> sum;
    {
      const uint4* at = mine;
      if (half > 0) cp_async_wait<1>();
      for (int g = 0; g < whole; ++g, at += kStep) {
        if (g == half) cp_async_wait<0>();
        uint4 u[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) u[j] = at[j * T];
        sum.add(u, c);
      }
      if (whole == 0) cp_async_wait<0>();
#pragma unroll 1
      for (int v = rest; v < nv; v += T) {
        const uint4 u[1] = {cut(ring[v], v, valid)};
        sum.add(u, c);
      }
    }
    sum.leave(c, red[parity]);
    bar_sync(kSums, T + 32);
    sum.join(c, red[parity], T >> 5);
    const Weights w = weights_of<K>(a, sum.m, sum.soft, sum.hard, has[parity] != 0, labels[parity] >= 0);
    // (rows that nothing is learnt from get zeros, whatever their logits are)
    const bool learnt = w.drop != 0.f || w.label != 0.f, more = row + (int)gridDim.x < a.rows;
    const uint4* z = logits_row(more ? row + gridDim.x : row);
    uint4* out = reinterpret_cast<uint4*>(out_row(row));
    {
      const uint4 *at = mine, *next = z + threadIdx.x;
      uint4* to = out + threadIdx.x;
      for (int g = 0; g < whole; ++g, at += kStep, to += kStep, next += kStep) {
        if (learnt) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) to[j * T] = grad_whole<K>(at[j * T], w);
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) to[j * T] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (g == 0) bar_sync(kTaken, T + 32);      // the clerk has what it wants of this row
        if (more) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) cp_async16(const_cast<uint4*>(at) + j * T, next + j * T);
        }
        if (g + 1 == half) cp_async_commit();
      }
    }
    if (whole == 0) bar_sync(kTaken, T + 32);
#pragma unroll 1
    for (int v = rest; v < nv; v += T) {
      out[v] = learnt ? grad_vector<K>(ring[v], v, valid, w) : make_uint4(0u, 0u, 0u, 0u);
      if (more) cp_async16(ring + v, z + v);
    }
    cp_async_commit();
    for (int v = nv + threadIdx.x; v < nvec; v += T) out[v] = make_uint4(0u, 0u, 0u, 0u);
    bar_arrive(kWritten, T + 32);
  }
}

// Of sums relative to 2^ref, relative to 2^(m c): times 2^(ref - m c), whose exponent fma gives exactly.
__device__ __forceinline__ float shift(float m, float c) { return near(ref_of(m, c)) ? exp2f(fmaf(-m, c, ref_of(m, c))) : 1.f; }
// sum p (z - m) over the entries, from the sum of p z: of logits whose differences are far below their size, what the sums' rounding
// (2^-18 of it: up to 1024 entries in fp32) cannot tell from 0 is 0.
__device__ __forceinline__ float above(float dot, float total, float m, float c) {
  const float d = dot - total * m;
  return !near(ref_of(m, c)) && fabsf(d) <= fminf(fabsf(m), FLT_MAX) * 3.814697265625e-6f ? 0.f : d;
}

// Statistics of a slice.
__global__ void __launch_bounds__(512)
distill_partial_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 ring[];
  __shared__ float red[96];
  const int T = blockDim.x, row = blockIdx.x, valid = max(0, min(a.cols, a.vocab - a.col_offset)), nv = (valid + 7) >> 3;
  const float c = kLog2e / a.temperature;
  const __nv_bfloat16* z = reinterpret_cast<const __nv_bfloat16*>(a.logits) + (int64_t)row * a.ld;
  const uint4* zv = reinterpret_cast<const uint4*>(z);
  grid_trigger();
  grid_wait();
  Sums<kTwo> sum;
  for (int v0 = threadIdx.x; v0 < nv; v0 += T * kVec) {
    uint4 u[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int v = v0 + j * T;
      u[j] = v < nv ? cut(zv[v], v, valid) : make_uint4(kNegInf2, kNegInf2, kNegInf2, kNegInf2);
    }
    sum.add(u, c);
  }
  sum.leave(c, red);
  __syncthreads();
  if (threadIdx.x < 32) {
    sum.join(c, red, T >> 5);
    const Entries raw = entries_at(ring, a.top), e = entries_at(reinterpret_cast<uint8_t*>(ring) + entry_bytes(a.top), a.top);
    const RowTarget t = read_entries(a, row, hold(a, row), raw, e);
    float dot = 0.f;
    for (int k = threadIdx.x; k <= a.top; k += 32) {
      const int at = e.at[k] - a.col_offset;
      if (e.at[k] >= 0 && at >= 0 && at < valid && e.p[k] != 0.f) dot += e.p[k] * __bfloat162float(z[at]);
    }
    dot = warp_sum(dot);
    if (threadIdx.x == 0) {
      const int y = t.label - a.col_offset;
      float* s = a.stats + (int64_t)row * 5;
      s[0] = sum.m;
      s[1] = sum.hard * shift(sum.m, kLog2e);       // relative to the maximum itself
      s[2] = sum.soft * shift(sum.m, c);
      s[3] = dot;
      s[4] = t.label >= 0 && y >= 0 && y < valid ? __bfloat162float(z[y]) : 0.f;
    }
  }
}

// Gradient of a slice from the statistics of whole rows.
template <int K>
__global__ void __launch_bounds__(512)
distill_grad_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 ring[];
  __shared__ RowTarget target;
  const int T = blockDim.x, row = blockIdx.x, nvec = a.cols >> 3, valid = max(0, min(a.cols, a.vocab - a.col_offset));
  const float c = kLog2e / a.temperature;
  const __nv_bfloat16* z = reinterpret_cast<const __nv_bfloat16*>(a.logits) + (int64_t)row * a.ld;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.grad) + (int64_t)row * a.ldg;
  const Entries raw = entries_at(ring, a.top), e = entries_at(reinterpret_cast<uint8_t*>(ring) + entry_bytes(a.top), a.top);
  grid_trigger();
  grid_wait();
  const float* s = a.stats + (int64_t)row * 5;
  const float m = s[0], hard = s[1], soft = s[2];
  if (threadIdx.x < 32) {
    const RowTarget t = read_entries(a, row, hold(a, row), raw, e);
    float total = 0.f;
    for (int k = threadIdx.x; k <= a.top; k += 32) total += e.at[k] >= 0 ? e.p[k] : 0.f;
    total = warp_sum(total);
    if (threadIdx.x == 0) {
      target = t;
      if (a.loss != nullptr) a.loss[row] = loss_of(a, t, soft, hard, above(s[3], total, m, c) / a.temperature, total, s[4] - m);
    }
  }
  __syncthreads();
  const Weights w = weights_of<K>(a, m, soft / shift(m, c), hard / (powers(K) > 1 ? powf(shift(m, c), powers(K)) : shift(m, kLog2e)),
                                  target.some, target.label >= 0);
  for (int k = threadIdx.x; k <= a.top; k += T) {          // before the gradient may overwrite the logits
    const int at = e.at[k] - a.col_offset;
    const bool here = e.at[k] >= 0 && at >= 0 && at < valid;
    const float drop = here ? drop_of(w, e.at[k], e.p[k], target.label) : 0.f;
    if (drop != 0.f) e.p[k] = grad_one<K>(__bfloat162float(z[at]), w) - drop;
    else e.at[k] = -1;
  }
  __syncthreads();
  const int learnt = w.drop == 0.f && w.label == 0.f ? 0 : (valid + 7) >> 3;
  for (int v0 = threadIdx.x; v0 < nvec; v0 += T * kVec) {
    uint4 u[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (v0 + j * T < learnt) u[j] = reinterpret_cast<const uint4*>(z)[v0 + j * T];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int v = v0 + j * T;
      if (v < nvec) reinterpret_cast<uint4*>(out)[v] = v < learnt ? grad_vector<K>(u[j], v, valid, w) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k <= a.top; k += T)
    if (e.at[k] >= 0) out[e.at[k] - a.col_offset] = __float2bfloat16(e.p[k]);
}

cudaError_t check(const DistillArgs& a) {
  const auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (a.rows <= 0 || a.cols <= 0 || a.cols % 8 || a.vocab <= 0 || a.col_offset < 0 || a.top < 0 || a.top > kDistillTop)
    return cudaErrorInvalidValue;
  if (off(a.logits) || a.ld % 8 || a.ld < a.cols) return cudaErrorInvalidValue;
  if (!(a.temperature > 0.f) || !(a.hard >= 0.f && a.hard <= 1.f)) return cudaErrorInvalidValue;
  return cudaSuccess;
}
cudaError_t check_grad(const DistillArgs& a) {
  return (reinterpret_cast<uintptr_t>(a.grad) & 15) || a.ldg % 8 || a.ldg < a.cols ? cudaErrorInvalidValue : check(a);
}
int kind_of(const DistillArgs& a) {
  if (a.hard == 0.f || a.temperature == 1.f) return kSoft;
  return a.hard == 1.f ? kHard : a.temperature == 2.f ? kSquare : a.temperature == 4.f ? kFourth : kTwo;
}
template <class Kernel>
cudaError_t allow(Kernel kernel, int bytes) {
  return bytes <= 31 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace

int distill_row_cols() { return kRowBytes / 2; }

cudaError_t distill_row(const DistillArgs& a, cudaStream_t stream) {
  cudaError_t e = check_grad(a);
  const int valid = a.cols < a.vocab ? a.cols : a.vocab, nv = (valid + 7) / 8;
  if (e != cudaSuccess) return e;
  if (valid > distill_row_cols() || a.col_offset != 0 || a.cols < a.vocab) return cudaErrorInvalidValue;
  const int smem = nv * 16 + 3 * entry_bytes(a.top), kind = kind_of(a);
  // As many CTAs as are resident at a time: by shared memory (228 KiB, 2 KiB a CTA beside the row) and registers.
  static int counts[64] = {0};
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) {
    if (counts[dev] == 0 && cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) counts[dev] = 148;
    sms = counts[dev];
  }
  const int fit = 228 * 1024 / (smem + 2048), T = fit < 2 ? 512 : nv > 1024 ? 256 : 128;
  const auto of_kind = [&](auto width) {
    constexpr int W = decltype(width)::value;
    return kind == kSoft ? distill_row_kernel<kSoft, W> : kind == kHard ? distill_row_kernel<kHard, W>
         : kind == kSquare ? distill_row_kernel<kSquare, W> : kind == kFourth ? distill_row_kernel<kFourth, W> : distill_row_kernel<kTwo, W>;
  };
  auto kernel = T == 512 ? of_kind(std::integral_constant<int, 512>()) : T == 256 ? of_kind(std::integral_constant<int, 256>())
                                                                                 : of_kind(std::integral_constant<int, 128>());
  e = allow(kernel, smem);
  if (e != cudaSuccess) return e;
  const int64_t most = (int64_t)sms * (fit < 1 ? 1 : fit < row_ctas(T) ? fit : row_ctas(T));
  return launch_dependent(kernel, (unsigned)(a.rows < most ? a.rows : most), T + 32, smem, stream, a);
}
cudaError_t distill_partial(const DistillArgs& a, cudaStream_t stream) {
  const cudaError_t e = check(a);
  if (e != cudaSuccess) return e;
  return launch_dependent(distill_partial_kernel, a.rows, 512, 2 * entry_bytes(a.top), stream, a);
}
cudaError_t distill_grad(const DistillArgs& a, cudaStream_t stream) {
  const cudaError_t e = check_grad(a);
  if (e != cudaSuccess) return e;
  const int kind = kind_of(a);
  auto kernel = kind == kSoft ? distill_grad_kernel<kSoft> : kind == kHard ? distill_grad_kernel<kHard>
              : kind == kSquare ? distill_grad_kernel<kSquare> : kind == kFourth ? distill_grad_kernel<kFourth> : distill_grad_kernel<kTwo>;
  return launch_dependent(kernel, a.rows, 512, 2 * entry_bytes(a.top), stream, a);
}

}  // namespace msb
