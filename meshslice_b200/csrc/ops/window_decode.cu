// Attention of single tokens over the ring cache of a windowed model.
#include "window_decode.h"

#include <cuda_bf16.h>
#include <math.h>

#include "../common/pdl.cuh"
#include "../common/ptx.cuh"

namespace msb {

namespace {

constexpr int kD = 128;
constexpr int kWarps = 4;
constexpr int kKeys = 16;                          // slots of a tile: one warp's step
constexpr int kTile = kKeys * kD * 2;              // 4 KiB, of K or of V
constexpr int kStages = 3;
constexpr int kHeads = 16;                         // query heads of a CTA: rows of a matrix fragment
constexpr int kSmem = kWarps * kStages * 2 * kTile;
constexpr int kPart = kWindowDecodePart;           // floats of a split: O, m, l
static_assert(kPart == kHeads * (kD + 2), "what a split leaves");
constexpr int kClusterSplits = kWindowDecodeCluster;
constexpr float kLog2e = 1.4426950408889634f;
static_assert(kWarps * kHeads * (kD + 2) * 4 <= kSmem, "the warps' results take the place of the tiles");

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  // what is not there is filled with zeros: the cache may hold anything beyond the last position
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A maximum to subtract: where all scores so far are -inf, -inf - 0 gives the probability 0 that -inf + inf would not.
__device__ __forceinline__ float finite(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ uint32_t pack(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8]
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t of_rank(uint32_t at, int rank) {       // the same place of another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ float load_of(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 load4_of(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
// What the CTAs of the cluster that have not left wrote to their shared memory before this is seen after it.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// A CTA works on a run of slots of one (sequence, key/value head, 16 of its query heads); each warp on every fourth tile of 16
// slots, with running maximum and sum of its own, through a ring that it fills itself (cp.async; no barrier).  The query heads
// are the rows of the matrix fragments, so that all heads of a group share a pass over K and V.  mma.sync: a token's products are a
// sixth of what that path does beside the memory, and the operands come as rows of any number and origin.
// The token's own k and v are taken from `qkv` in place of their slot, which the CTA that has it writes.
// Splits of a sequence are joined in their order: up to 8 are a cluster, whose CTAs take the heads by turns from the shared memory of
// all, more by the CTA that finishes last, through memory.  P is rounded to bf16 as the operand of P V.
// Bound by HBM: 64 sequences of up to 4100 slots, 8 x 4 heads, 145 us (6.6 TB/s); one sequence of 700 tokens by the launch and two
// trips to memory (position, tiles): 6.7 us (8.2 where its splits were joined through memory).
// kWide: more than 8 query heads (rows 8 to 15 of the fragments are in use).
// kCluster: the splits of a sequence are a cluster, and each CTA joins some of its heads from the shared memory of all.
template <bool kWide, bool kCluster>
__global__ void __launch_bounds__(kWarps * 32)
window_decode_kernel(const __grid_constant__ WindowDecodeArgs a, int splits, int per_split) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int passes = (a.group + kHeads - 1) / kHeads;
  const int split = blockIdx.x, h = blockIdx.y / passes, g0 = (blockIdx.y - h * passes) * kHeads, b = blockIdx.z;
  const int heads = min(kHeads, a.group - g0), slots = a.sinks + a.window;
  grid_trigger();
  grid_wait();
  const int64_t pos = a.positions[b];
  const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(a.qkv) + b * a.ld + (int64_t)h * (a.group + 2) * kD;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + ((int64_t)(b * a.kv + h) * a.group + g0) * kD;
  if (pos < 0) {
    if (split == 0)
      for (int i = threadIdx.x; i < heads * kD / 8; i += kWarps * 32) reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const int held = pos < slots ? (int)pos + 1 : slots;
  const int own = pos < a.sinks ? (int)pos : a.sinks + (int)(pos < 1ll << 31 ? (uint32_t)(pos - a.sinks) % (uint32_t)a.window : (pos - a.sinks) % a.window);
  const int s0 = split * per_split, s1 = min(held, s0 + per_split);
  if (s0 >= held) return;
  const int64_t base = ((int64_t)b * a.kv + h) * slots * kD;
  __nv_bfloat16 *ck = reinterpret_cast<__nv_bfloat16*>(a.k) + base, *cv = reinterpret_cast<__nv_bfloat16*>(a.v) + base;
  const __nv_bfloat16 *nk = row + a.group * kD, *nv = nk + kD;
  if (g0 == 0 && own >= s0 && own < s1 && threadIdx.x < 32) {
    const int i = threadIdx.x & 15;
    const uint4 u = reinterpret_cast<const uint4*>(threadIdx.x < 16 ? nk : nv)[i];
    reinterpret_cast<uint4*>((threadIdx.x < 16 ? ck : cv) + (int64_t)own * kD)[i] = u;
  }

  const int tiles = (s1 - s0 + kKeys - 1) / kKeys;
  const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * kTile;
  auto fetch = [&](int tile, int stage) {
    if (tile < tiles) {
      const uint32_t at = ring + stage * 2 * kTile;
      // 16 lanes a row; chunk c of row r lies at c ^ (r % 8): fragments are read without conflicts
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 2 + (lane >> 4), c = lane & 15, slot = s0 + tile * kKeys + r;
        const bool there = slot < s1;
        const int64_t off = (int64_t)(there ? slot : s0) * kD + c * 8;
        const uint32_t to = at + r * 256 + ((c ^ (r & 7)) << 4);
        copy16(to, slot == own ? nk + c * 8 : ck + off, there);
        copy16(to + kTile, slot == own ? nv + c * 8 : cv + off, there);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(warp + i * kWarps, i);
  // query heads as A fragments: rows lane / 4 and + 8, columns 2 (lane % 4) and + 8 of each 16
  uint32_t q[8][4];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + (i & 1) * 8, col = ks * 16 + (i >> 1) * 8 + (lane & 3) * 2;
      q[ks][i] = (kWide || !(i & 1)) && r < heads ? *reinterpret_cast<const uint32_t*>(row + (g0 + r) * kD + col) : 0u;
    }
  float o[16][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float sl2 = a.scale * kLog2e;
  int stage = 0;
  for (int tile = warp; tile < tiles; tile += kWarps) {
    fetch(tile + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1);
    copy_wait<kStages - 1>();
    __syncwarp();
    const uint32_t at = ring + stage * 2 * kTile;
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t kb[4];
      const int r = (lane & 7) + (lane >> 4) * 8, c = ks * 2 + ((lane >> 3) & 1);
      load4(kb, at + r * 256 + ((c ^ (r & 7)) << 4));
      mma(s[0], q[ks], kb[0], kb[1]);
      mma(s[1], q[ks], kb[2], kb[3]);
    }
    // scores in the log2 domain; slots beyond the last one see nothing
    const int left = s1 - s0 - tile * kKeys;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = n * 8 + (lane & 3) * 2 + (i & 1);
        s[n][i] = key < left ? s[n][i] * sl2 : -INFINITY;
      }
    float up[2];
    bool grown = false;
#pragma unroll
    for (int r = 0; r < (kWide ? 2 : 1); ++r) {
      float t = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
      up[r] = fmaxf(m[r], t);
      grown |= up[r] > m[r];
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int r = 0; r < (kWide ? 2 : 1); ++r) {
        const float f = up[r] > m[r] ? exp2_ftz(m[r] - up[r]) : 1.f;
        l[r] *= f;
        m[r] = up[r];
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          o[n][2 * r] *= f;
          o[n][2 * r + 1] *= f;
        }
      }
    }
    uint32_t p[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < (kWide ? 2 : 1); ++r) {
        const float at = finite(m[r]), x = exp2_ftz(s[n][2 * r] - at), y = exp2_ftz(s[n][2 * r + 1] - at);
        l[r] += x + y;
        p[n * 2 + r] = pack(x, y);
      }
#pragma unroll
    for (int c = 0; c < 16; c += 2) {
      uint32_t vb[4];
      const int r = lane & 15, cc = c + (lane >> 4);
      load4_trans(vb, at + kTile + r * 256 + ((cc ^ (r & 7)) << 4));
      mma(o[c], p, vb[0], vb[1]);
      mma(o[c + 1], p, vb[2], vb[3]);
    }
    __syncwarp();                                  // the stage has been read
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  copy_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  // the warps' results: O [warp][head][128], m and l [warp][head]
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);
  float *sm = so + kWarps * kHeads * kD, *sl = sm + kWarps * kHeads;
#pragma unroll
  for (int r = 0; r < (kWide ? 2 : 1); ++r) {
    const int head = (lane >> 2) + r * 8;
    float* to = so + (warp * kHeads + head) * kD + (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < 16; ++n) *reinterpret_cast<float2*>(to + n * 8) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
    if ((lane & 3) == 0) {
      sm[warp * kHeads + head] = m[r];
      sl[warp * kHeads + head] = l[r];
    }
  }
  __syncthreads();
  // A warp a head from here on, four features a lane.
  const int live = (held + per_split - 1) / per_split;
  const int64_t unit = (int64_t)b * gridDim.y + blockIdx.y;
  const auto store = [&](int head, const float4& v, float by) {
    *reinterpret_cast<uint2*>(out + head * kD + lane * 4) = make_uint2(pack(v.x * by, v.y * by), pack(v.z * by, v.w * by));
  };
  const auto add = [](float4& acc, float f, const float4& v) {
    acc.x += f * v.x;
    acc.y += f * v.y;
    acc.z += f * v.z;
    acc.w += f * v.w;
  };
  float* part = a.parts + (unit * splits + split) * kPart;
  for (int head = warp; head < heads; head += kWarps) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w * kHeads + head]);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = w < tiles ? exp2_ftz(sm[w * kHeads + head] - finite(top)) : 0.f;            // a warp without a tile has nothing
      sum += f * sl[w * kHeads + head];
      add(acc, f, *reinterpret_cast<const float4*>(so + (w * kHeads + head) * kD + lane * 4));
    }
    if (live == 1) {
      store(head, acc, 1.f / sum);
    } else if constexpr (kCluster) {
      __syncwarp();
      *reinterpret_cast<float4*>(so + head * kD + lane * 4) = acc;                       // (read by this warp alone)
      if (lane == 0) {
        sm[head] = top;
        sl[head] = sum;
      }
    } else {
      __stcg(reinterpret_cast<float4*>(part + head * kD + lane * 4), acc);
      if (lane == 0) __stcg(reinterpret_cast<float2*>(part + kHeads * kD + head * 2), make_float2(top, sum));
    }
  }
  if (live == 1) return;                           // (CTAs without a slot have left: the barriers do not count them)
  if constexpr (kCluster) {
    cluster_barrier();
    const uint32_t at_o = smem_u32(so), at_m = smem_u32(sm), at_l = smem_u32(sl);
    for (int head = warp * live + split; head < heads; head += kWarps * live) {
      const int rank = min(lane, live - 1);
      const float m1 = load_of(of_rank(at_m + head * 4, rank)), l1 = load_of(of_rank(at_l + head * 4, rank));
      float4 v[kClusterSplits];
#pragma unroll
      for (int s = 0; s < kClusterSplits; ++s) v[s] = load4_of(of_rank(at_o + head * (kD * 4) + lane * 16, min(s, live - 1)));
      float t = m1;
#pragma unroll
      for (int o = kClusterSplits / 2; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
      const float f = lane < live ? exp2_ftz(m1 - finite(t)) : 0.f;
      float sum = f * l1;
#pragma unroll
      for (int o = kClusterSplits / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kClusterSplits; ++s)
        if (s < live) add(acc, __shfl_sync(0xffffffffu, f, s), v[s]);
      store(head, acc, 1.f / __shfl_sync(0xffffffffu, sum, 0));
    }
    cluster_barrier();                             // until here the others read this CTA's memory
    return;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = atomicAdd(a.counters + unit, 1u);
    last = before + 1 == (uint32_t)live;
    if (last) a.counters[unit] = 0;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  // The CTA that finishes last joins them, in their order: a lane has the statistics of every 32nd split.
  const float* parts = a.parts + unit * splits * kPart;
  const auto stats = [&](int s, int head) {
    return s < live ? __ldcg(reinterpret_cast<const float2*>(parts + s * kPart + kHeads * kD + head * 2)) : make_float2(-INFINITY, 0.f);
  };
  // (the heads of a warp together: their splits are on their way at the same time)
  constexpr int kEach = (kWide ? kHeads : 8) / kWarps;
  float top[kEach], sum[kEach];
  float4 acc[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int head = min(warp + i * kWarps, heads - 1);
    float t = -INFINITY;
    for (int s = lane; s < live; s += 32) t = fmaxf(t, stats(s, head).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    top[i] = t;
    sum[i] = 0.f;
    acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int s0 = 0; s0 < live; s0 += 32) {
    float f[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const float2 st = stats(s0 + lane, min(warp + i * kWarps, heads - 1));
      f[i] = s0 + lane < live ? exp2_ftz(st.x - finite(top[i])) : 0.f;
      sum[i] += f[i] * st.y;
    }
    const int n = min(32, live - s0);
    const float* from = parts + (int64_t)s0 * kPart + lane * 4;
#pragma unroll 4
    for (int s = 0; s < n; ++s)
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        add(acc[i], __shfl_sync(0xffffffffu, f[i], s),
            __ldcg(reinterpret_cast<const float4*>(from + (int64_t)s * kPart + min(warp + i * kWarps, heads - 1) * kD)));
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    float t = sum[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (warp + i * kWarps < heads) store(warp + i * kWarps, acc[i], 1.f / t);
  }
}

}  // namespace

// One wave of two CTAs an SM, in clusters of up to 8 with a tile or more for every warp.  A wide launch of long caches goes beyond a
// cluster: s splits cost slots / s for the tiles and s for the join through memory, least at a multiple of the root of slots.  us by splits:
// 64 sequences of 8 key heads, 4100 slots, 1 143, 2 155, 6 167; 256 of 8, 512 slots, 1 87, 2 118; 16 of 8, 4100, 1 56, 2 48, 4 49, 8 58; 1 of 8,
// 128 slots, 1 4.4, 2 4.8; 260, 1 5.7, 2 6.3, 5 5.0; 1028, 1 9.3, 4 8.3, 8 6.7, 12 9.0; 8196, 8 18.3, 18 16.6, 37 17.8; 65536, 8 106, 18 57, 24 52,
// 37 54; 3 of 8, 65536, 8 124, 12 130, 24 130; 1 of 1, 4096, 8 10.6, 12 14.3, 22 13.9; 8192, 8 15.8, 18 15.7, 43 20; 131072, 8 186, 37 45, 74 35, 148 40,
// 296 61.
int window_decode_splits(int batch, int kv, int group, int slots, int sms) {
  if (batch <= 0 || kv <= 0 || group <= 0 || slots <= 0 || sms <= 0) return 1;      // (nothing to deal out; such a launch is refused)
  const int64_t units = (int64_t)batch * kv * ((group + kHeads - 1) / kHeads), want = (int64_t)sms * 2 / units;
  const int tiles = kWarps * kKeys, most = slots <= 2 * tiles ? 1 : (slots + tiles - 1) / tiles;
  const int64_t wide = (int64_t)sqrt(slots / 24.);
  if (want >= 2 * kClusterSplits && wide >= 2 * kClusterSplits) return (int)(want < wide ? want : wide);
  const int64_t n = want < kClusterSplits ? want : kClusterSplits;
  return (int)(n < 1 ? 1 : n < most ? n : most);
}

cudaError_t window_decode(const WindowDecodeArgs& a, int splits, cudaStream_t stream) {
  const auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (a.batch <= 0 || a.kv <= 0 || a.group <= 0 || a.window <= 0 || a.sinks < 0 || splits <= 0) return cudaErrorInvalidValue;
  if (off(a.qkv) || off(a.k) || off(a.v) || off(a.out) || a.ld % 8) return cudaErrorInvalidValue;
  const int64_t slots = (int64_t)a.sinks + a.window, rows = (int64_t)a.kv * ((a.group + kHeads - 1) / kHeads);
  if (slots > 1 << 30 || rows > 65535 || a.batch > 65535) return cudaErrorInvalidValue;
  const int steps = kWarps * kKeys, per = (int)((slots + splits - 1) / splits + steps - 1) / steps * steps;
  if (splits > kClusterSplits && (a.parts == nullptr || off(a.parts) || a.counters == nullptr)) return cudaErrorInvalidValue;
  const bool wide = a.group > 8, cluster = splits > 1 && splits <= kClusterSplits;
  auto kernel = wide ? cluster ? window_decode_kernel<true, true> : window_decode_kernel<true, false>
                     : cluster ? window_decode_kernel<false, true> : window_decode_kernel<false, false>;
  // the attribute is per device: set it once on every device that launches
  static bool configured[64][4] = {};
  const int which = wide * 2 + cluster;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev][which]) {
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev][which] = true;
  }
  return launch_dependent_clusters(kernel, cluster ? splits : 1, dim3((unsigned)splits, (unsigned)rows, (unsigned)a.batch), kWarps * 32, kSmem, stream, a, splits, per);
}

}  // namespace msb
