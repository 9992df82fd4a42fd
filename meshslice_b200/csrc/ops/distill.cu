// Distillation loss over rows of logits: softmax statistics, the teacher's few entries, the gradient.
#include "distill.h"

#include <cuda_bf16.h>

#include "../common/f32x2.cuh"
#include "../common/pdl.cuh"
#include "../common/ptx.cuh"

namespace msb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kNegInf2 = 0xff80ff80u;       // two bf16 -inf
constexpr int kVec = 4;                          // vectors of a thread that are worked on together
constexpr int kAhead = 4;                        // groups of kVec that are on their way
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

// Which exponentials a row needs: those of z / T, of z, or both (one kind serves both where T = 1).
enum Kind { kSoft = 1, kHard = 2, kTwo = 3 };

// A thread's running maximum m, and sums of exp(z - m) and exp((z - m) / T).  Differences are taken first: they are exact where they
// matter, and a rounded m / T would shift the whole row.
template <int K>
struct Sums {
  float m = -INFINITY, soft = 0.f, hard = 0.f;
  __device__ __forceinline__ void raise(float to, float c) {
    if (to > m) {
      if (K & kSoft) soft *= exp2_ftz((m - to) * c);      // (0 while m is -inf: the sums are 0)
      if (K & kHard) hard *= exp2_ftz((m - to) * kLog2e);
      m = to;
    }
  }
  __device__ __forceinline__ void add(const uint4 (&u)[kVec], float c) {
    uint32_t top = kNegInf2;
#pragma unroll
    for (int j = 0; j < kVec; ++j) top = max_bf16x2(max_bf16x2(max_bf16x2(top, u[j].x), max_bf16x2(u[j].y, u[j].z)), u[j].w);
    raise(fmaxf(lo(top), hi(top)), c);
    if (m > -INFINITY) {
      const uint64_t neg_m = both(-m), cs = both(c), ch = both(kLog2e);
      uint64_t ps[kVec] = {}, ph[kVec] = {};
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t d = add2(unpack2(w[i]), neg_m);
          float a, b;
          if (K & kSoft) {
            split(mul2(d, cs), a, b);
            ps[j] = add2(ps[j], f32x2(exp2_ftz(a), exp2_ftz(b)));
          }
          if (K & kHard) {
            split(mul2(d, ch), a, b);
            ph[j] = add2(ph[j], f32x2(exp2_ftz(a), exp2_ftz(b)));
          }
        }
      }
      float a, b;
      if (K & kSoft) {
        split(add2(add2(ps[0], ps[1]), add2(ps[2], ps[3])), a, b);
        soft += a + b;
      }
      if (K & kHard) {
        split(add2(add2(ph[0], ph[1]), add2(ph[2], ph[3])), a, b);
        hard += a + b;
      }
    } else {
      // while everything seen is -inf nothing counts, except that a NaN has to show
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = lo(w[i]), b = hi(w[i]), n = (a == a ? 0.f : a) + (b == b ? 0.f : b);
          soft += n;
          hard += n;
        }
      }
    }
  }
  // Maximum and sums of the CTA, for every thread.  red: 3 * 32 floats.
  __device__ __forceinline__ void block(float c, float* red) {
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31, nw = blockDim.x >> 5;
    // (a warp of threads without an element has sums of 0, or NaN)
    const float mw = warp_max(m);
    const float s = m == -INFINITY && mw > -INFINITY ? soft : soft * exp2_ftz((m - mw) * c);
    const float h = m == -INFINITY && mw > -INFINITY ? hard : hard * exp2_ftz((m - mw) * kLog2e);
    soft = warp_sum(mw == -INFINITY ? soft : s);
    hard = warp_sum(mw == -INFINITY ? hard : h);
    __syncthreads();
    if (l == 0) { red[w] = mw; red[32 + w] = soft; red[64 + w] = hard; }
    __syncthreads();
    const float mine = l < nw ? red[l] : -INFINITY;
    m = warp_max(mine);
    soft = l < nw ? red[32 + l] : 0.f;
    hard = l < nw ? red[64 + l] : 0.f;
    if (mine > -INFINITY) {
      soft *= exp2_ftz((mine - m) * c);
      hard *= exp2_ftz((mine - m) * kLog2e);
    }
    soft = warp_sum(soft);
    hard = warp_sum(hard);
  }
};

// The teacher's entries of a row in shared memory: id - col_offset, or -1 for no entry; probability.  Entry `top` is the label.
struct Entries {
  int* id;
  float* p;
};
__host__ __device__ constexpr int entry_bytes(int top) { return (top + 1 + 3) / 4 * 4 * 8; }
__device__ __forceinline__ Entries entries_at(void* at, int top) {
  Entries e;
  e.id = reinterpret_cast<int*>(at);
  e.p = reinterpret_cast<float*>(e.id + (top + 1 + 3) / 4 * 4);
  return e;
}
__device__ __forceinline__ float value_at(const DistillArgs& a, int64_t i) {
  return a.values_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.values)[i]) : reinterpret_cast<const float*>(a.values)[i];
}
// By one warp.  Returns whether the row has an entry of any weight, and sum p log p.
__device__ __forceinline__ bool read_entries(const DistillArgs& a, int row, const Entries& e, float& plogp) {
  const int l = threadIdx.x & 31;
  const int64_t base = (int64_t)row * a.top;
  const float c = kLog2e / a.temperature;
  float mx = -INFINITY;
  for (int k = l; k < a.top; k += 32) {
    const int64_t id = a.ids[base + k];
    const bool there = id >= 0 && id < a.vocab;
    const float v = there ? value_at(a, base + k) : -INFINITY;
    e.id[k] = there ? (int)id : -1;
    e.p[k] = v;
    mx = v > mx || v != v ? v : mx;
  }
  mx = warp_max(mx);
  float sum = 0.f;
  for (int k = l; k < a.top; k += 32) {
    const float x = e.p[k] == -INFINITY ? 0.f : exp2_ftz((e.p[k] - mx) * c);
    sum += x;
    e.p[k] = x;
  }
  sum = warp_sum(sum);
  plogp = 0.f;
  for (int k = l; k < a.top; k += 32) {
    const float p = sum == 0.f ? 0.f : e.p[k] / sum;
    if (p != 0.f) plogp += p * logf(p);
    e.p[k] = p;
  }
  plogp = warp_sum(plogp);
  if (l == 0) {
    const int64_t y = a.targets != nullptr ? a.targets[row] : -1;
    e.id[a.top] = y >= 0 && y < a.vocab ? (int)y : -1;
    e.p[a.top] = 0.f;
  }
  __syncwarp();
  return sum != 0.f;
}

// What the gradient of a row is made of: soft * exp((z - m) / T) + hard * exp(z - m), less `drop` times an entry's probability and
// `label` at the label.
struct Weights {
  float m, soft, hard, drop, label;
};
__device__ __forceinline__ Weights weights_of(const DistillArgs& a, float m, float soft, float hard, bool some, bool label) {
  Weights w;
  w.m = m;
  w.drop = some ? (1.f - a.hard) * a.temperature * a.scale : 0.f;
  w.label = label ? a.hard * a.scale : 0.f;
  w.soft = w.drop / soft;
  w.hard = w.label / hard;
  return w;
}
template <int K>
__device__ __forceinline__ uint32_t grad_pair(uint32_t z, const Weights& w, float c) {
  const uint64_t d = add2(unpack2(z), both(-w.m));
  float a, b;
  uint64_t g = 0;
  if (K & kSoft) {
    split(mul2(d, both(c)), a, b);
    g = mul2(f32x2(exp2_ftz(a), exp2_ftz(b)), both(w.soft));
  }
  if (K & kHard) {
    split(mul2(d, both(kLog2e)), a, b);
    g = fma2(f32x2(exp2_ftz(a), exp2_ftz(b)), both(w.hard), g);
  }
  split(g, a, b);
  return pack(a, b);
}
template <int K>
__device__ __forceinline__ float grad_one(float z, const Weights& w, float c) {
  float g = 0.f;
  if (K & kSoft) g = exp2_ftz((z - w.m) * c) * w.soft;
  if (K & kHard) g += exp2_ftz((z - w.m) * kLog2e) * w.hard;
  return g;
}
template <int K>
__device__ __forceinline__ uint4 grad_vector(uint4 u, int v, int valid, const Weights& w, float c) {
  // (rows that nothing is learnt from get zeros, whatever their logits are)
  if (v * 8 >= valid || (w.drop == 0.f && w.label == 0.f)) return make_uint4(0u, 0u, 0u, 0u);
  const uint4 g = make_uint4(grad_pair<K>(u.x, w, c), grad_pair<K>(u.y, w, c), grad_pair<K>(u.z, w, c), grad_pair<K>(u.w, w, c));
  if (v * 8 + 8 <= valid) return g;
  uint32_t r[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = v * 8 + 2 * i >= valid ? 0u : v * 8 + 2 * i + 1 >= valid ? r[i] & 0xffffu : r[i];
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// What entry k takes off its column's gradient; false where an earlier entry has the column (and takes it all).  In entry order.
__device__ __forceinline__ bool entry_drop(const Entries& e, int top, int k, const Weights& w, float& drop) {
  const int id = e.id[k];
  if (id < 0) return false;
  for (int j = 0; j < k; ++j)
    if (e.id[j] == id) return false;
  float p = 0.f;
  for (int j = k; j < top; ++j)
    if (e.id[j] == id) p += e.p[j];
  drop = w.drop * p + (e.id[top] == id ? w.label : 0.f);
  return true;
}
// A row's loss by one warp, from z of its entries.
template <class Z>
__device__ __forceinline__ float loss_of(const DistillArgs& a, const Entries& e, float m, float soft, float hard, bool some, float plogp, Z z) {
  float cross = 0.f;                       // sum p (z - m)
  for (int k = threadIdx.x & 31; k < a.top; k += 32)
    if (e.id[k] >= 0 && e.p[k] != 0.f) cross += e.p[k] * (z(e.id[k]) - m);
  cross = warp_sum(cross);
  float loss = 0.f;
  if (some && a.hard != 1.f) loss = (1.f - a.hard) * a.temperature * (a.temperature * (plogp + logf(soft)) - cross);
  if (e.id[a.top] >= 0 && a.hard != 0.f) loss += a.hard * (logf(hard) - (z(e.id[a.top]) - m));
  return loss;
}

// Whole rows: a row waits in shared memory between the sums and the gradient, so the logits are read once.
template <int K>
__global__ void __launch_bounds__(512)
distill_row_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 ring[];
  __shared__ float red[96];
  __shared__ int has;
  const int T = blockDim.x, row = blockIdx.x, nvec = a.cols >> 3, valid = min(a.cols, a.vocab), nv = (valid + 7) >> 3;
  const float c = kLog2e / a.temperature;
  const uint4* z = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.logits) + (int64_t)row * a.ld);
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.grad) + (int64_t)row * a.ldg;
  const Entries e = entries_at(ring + nv, a.top);
  grid_trigger();
  grid_wait();
  auto prefetch = [&](int v0) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int v = v0 + j * T;
      if (v < nv) cp_async16(ring + v, z + v);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) prefetch(threadIdx.x + i * T * kVec);
  float plogp = 0.f;
  if (threadIdx.x < 32) {
    const bool some = read_entries(a, row, e, plogp);
    if (threadIdx.x == 0) has = some;
  }
  Sums<K> sum;
  for (int v0 = threadIdx.x; v0 < nv; v0 += T * kVec) {
    prefetch(v0 + kAhead * T * kVec);
    cp_async_wait<kAhead>();
    uint4 u[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int v = v0 + j * T;
      u[j] = v < nv ? cut(ring[v], v, valid) : make_uint4(kNegInf2, kNegInf2, kNegInf2, kNegInf2);
    }
    sum.add(u, c);
  }
  cp_async_wait<0>();
  sum.block(c, red);                       // (its barriers make the row and its entries visible to every thread)
  if (K == kSoft) sum.hard = sum.soft;     // T = 1, or nothing of weight
  if (K == kHard) sum.soft = sum.hard;
  const bool some = has != 0;
  Weights w = weights_of(a, sum.m, sum.soft, sum.hard, some, e.id[a.top] >= 0);
  if (K == kSoft) w.soft += a.temperature == 1.f ? w.hard : 0.f;
  const __nv_bfloat16* kept = reinterpret_cast<const __nv_bfloat16*>(ring);
  for (int v = threadIdx.x; v < nvec; v += T)
    reinterpret_cast<uint4*>(out)[v] = grad_vector<K>(v < nv ? ring[v] : make_uint4(0u, 0u, 0u, 0u), v, valid, w, c);
  if (threadIdx.x < 32) {
    const float loss = loss_of(a, e, sum.m, sum.soft, sum.hard, some, plogp, [&](int id) { return __bfloat162float(kept[id]); });
    if (threadIdx.x == 0) a.loss[row] = loss;
  }
  __syncthreads();                         // the row's gradient is written: its entries' columns are written again
  for (int k = threadIdx.x; k <= a.top; k += T) {
    float drop;
    if (entry_drop(e, a.top, k, w, drop) && drop != 0.f)
      out[e.id[k]] = __float2bfloat16(grad_one<K>(__bfloat162float(kept[e.id[k]]), w, c) - drop);
  }
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
  const Entries e = entries_at(ring, a.top);
  grid_trigger();
  grid_wait();
  float plogp = 0.f;
  if (threadIdx.x < 32) read_entries(a, row, e, plogp);
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
  sum.block(c, red);
  if (threadIdx.x < 32) {
    float dot = 0.f;
    for (int k = threadIdx.x; k < a.top; k += 32) {
      const int id = e.id[k] - a.col_offset;
      if (e.id[k] >= 0 && id >= 0 && id < valid && e.p[k] != 0.f) dot += e.p[k] * __bfloat162float(z[id]);
    }
    dot = warp_sum(dot);
    if (threadIdx.x == 0) {
      const int y = e.id[a.top] - a.col_offset;
      float* s = a.stats + (int64_t)row * 5;
      s[0] = sum.m;
      s[1] = sum.hard;
      s[2] = sum.soft;
      s[3] = dot;
      s[4] = e.id[a.top] >= 0 && y >= 0 && y < valid ? __bfloat162float(z[y]) : 0.f;
    }
  }
}

// Gradient of a slice from the statistics of whole rows.
template <int K>
__global__ void __launch_bounds__(512)
distill_grad_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 ring[];
  __shared__ int has;
  const int T = blockDim.x, row = blockIdx.x, nvec = a.cols >> 3, valid = max(0, min(a.cols, a.vocab - a.col_offset));
  const float c = kLog2e / a.temperature;
  const __nv_bfloat16* z = reinterpret_cast<const __nv_bfloat16*>(a.logits) + (int64_t)row * a.ld;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.grad) + (int64_t)row * a.ldg;
  const Entries e = entries_at(ring, a.top);
  float* ze = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ring) + entry_bytes(a.top));   // z of the entries in this slice
  grid_trigger();
  grid_wait();
  const float* s = a.stats + (int64_t)row * 5;
  const float m = s[0], hard = s[1], soft = s[2];
  if (threadIdx.x < 32) {
    float plogp;
    const bool some = read_entries(a, row, e, plogp);
    float total = 0.f;
    for (int k = threadIdx.x; k < a.top; k += 32) total += e.p[k];
    total = warp_sum(total);
    if (threadIdx.x == 0) {
      has = some;
      if (a.loss != nullptr) {
        float loss = 0.f;
        if (some && a.hard != 1.f) loss = (1.f - a.hard) * a.temperature * (a.temperature * (plogp + logf(soft)) - (s[3] - total * m));
        if (e.id[a.top] >= 0 && a.hard != 0.f) loss += a.hard * (logf(hard) - (s[4] - m));
        a.loss[row] = loss;
      }
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k <= a.top; k += T) {          // before the gradient may overwrite the logits
    const int id = e.id[k] - a.col_offset;
    ze[k] = e.id[k] >= 0 && id >= 0 && id < valid ? __bfloat162float(z[id]) : 0.f;
  }
  __syncthreads();
  Weights w = weights_of(a, m, soft, hard, has != 0, e.id[a.top] >= 0);
  if (K == kSoft) w.soft += a.temperature == 1.f ? w.hard : 0.f;
  for (int v0 = threadIdx.x; v0 < nvec; v0 += T * kVec) {
    uint4 u[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (v0 + j * T < nvec) u[j] = reinterpret_cast<const uint4*>(z)[v0 + j * T];
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (v0 + j * T < nvec) reinterpret_cast<uint4*>(out)[v0 + j * T] = grad_vector<K>(u[j], v0 + j * T, valid, w, c);
  }
  __syncthreads();
  for (int k = threadIdx.x; k <= a.top; k += T) {
    const int id = e.id[k] - a.col_offset;
    float drop;
    if (e.id[k] >= 0 && id >= 0 && id < valid && entry_drop(e, a.top, k, w, drop) && drop != 0.f)
      out[id] = __float2bfloat16(grad_one<K>(ze[k], w, c) - drop);
  }
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
  return a.hard == 1.f ? kHard : kTwo;
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
  const int smem = nv * 16 + entry_bytes(a.top), kind = kind_of(a);
  auto kernel = kind == kSoft ? distill_row_kernel<kSoft> : kind == kHard ? distill_row_kernel<kHard> : distill_row_kernel<kTwo>;
  e = allow(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, a.rows, nv > 2048 ? 512 : 256, smem, stream, a);
}
cudaError_t distill_partial(const DistillArgs& a, cudaStream_t stream) {
  const cudaError_t e = check(a);
  if (e != cudaSuccess) return e;
  return launch_dependent(distill_partial_kernel, a.rows, 512, entry_bytes(a.top), stream, a);
}
cudaError_t distill_grad(const DistillArgs& a, cudaStream_t stream) {
  const cudaError_t e = check_grad(a);
  if (e != cudaSuccess) return e;
  const int kind = kind_of(a);
  auto kernel = kind == kSoft ? distill_grad_kernel<kSoft> : kind == kHard ? distill_grad_kernel<kHard> : distill_grad_kernel<kTwo>;
  return launch_dependent(kernel, a.rows, 512, entry_bytes(a.top) + 4 * (a.top + 1), stream, a);
}

}  // namespace msb
