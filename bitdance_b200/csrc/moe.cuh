// moe.cuh -- a mixture-of-experts layer for a few tokens (T <= 64) in two kernels, expert weights
// in NVFP4 as bd_quantize_b_nvfp4 writes them (natural codes and scales, nothing packed):
//
//   logits = x Wr^T;  s = softmax or sigmoid(logits);  top-k by s (+ bias);  w = s (renormalised)
//   y_t = sum over the chosen experts e of w_e * Wd_e (silu(Wg_e x_t) * (Wu_e x_t))
//
// A few tokens read far more weights than they compute with, so the experts' kernel streams
// the touched experts' 4-bit weights once, straight into registers, turns them into 16-bit MMA
// fragments there (exactly: an E2M1 times an E4M3 value has at most 6 significant bits) and
// multiplies by all tokens of the expert with mma.sync (weights are the 16 rows, tokens the 8
// columns; the tensor work is far below what the weights' bytes cost, and fragments in registers
// need no shared-memory staging). Activations are exact too: a token's values are scaled by a power
// of two into fp16 range by the first kernel. The hidden values (already times w and the down
// scale) are rounded once to bf16; sums are fp32.
//
// Kernel 1 (moe_route_kernel, or moe_prepare_kernel where the caller brings the routing): router
// products, selection, fp16 image of x, counters to zero.
// Kernel 2 (moe_experts_kernel): gate / up phase, then down phase in the same grid. Work is handed
// out by tickets (atomic counters), gate / up shares before down tasks: a CTA that waits for the
// hidden values knows that every share is held by a CTA that already runs, so the wait ends without
// any guarantee that the whole grid is resident at once.
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "epilogue.cuh"
#include "sm100.cuh"

namespace bd {

constexpr int kMoeMaxTokens = 64, kMoeMaxExperts = 512, kMoeMaxTopK = 16;
constexpr int kMoeThreads = 256, kMoeWarps = kMoeThreads / 32;
constexpr int kRouteCluster = 8;

enum : int { kMoeShares = 0, kMoeDone = 1, kMoeDown = 2, kMoeCounters = 3 };

// Position of element k of a row in the scratch images of x and h. A thread of an MMA lane quad q
// takes elements 32 q .. 32 q + 31 of a 128-block (one 16-byte piece of the weights' codes), in four
// loads of 8: load j of the quad is 64 contiguous bytes when (q, j) are exchanged.
__host__ __device__ __forceinline__ int moe_perm(int k) {
  const int r = k & 127;
  return (k & ~127) + ((r >> 3) & 3) * 32 + (r >> 5) * 8 + (r & 7);
}
// h besides pairs elements m and m + 4 of a group of 8 (the pairs one shift of a word of codes
// brings to the low ends of both 16-bit halves).
__host__ __device__ __forceinline__ int moe_perm_h(int k) {
  const int m = k & 7;
  return (moe_perm(k) & ~7) + (m < 4 ? 2 * m : 2 * (m - 4) + 1);
}

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// 8 consecutive elements as floats (16-byte aligned).
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(e[j]);
  }
}

// ---------------------------------------------------------------------------------- kernel 1

struct MoeRouteParams {
  const void* x;
  const void* router;      // (E, H)
  const float* bias;       // (E,) added for the selection only, may be null
  int* ids;                // (T, k)
  float* weights;          // (T, k)
  __half* xs;              // (T, H) fp16 image, permuted
  float* x_scale;          // (T,) power of two
  uint32_t* counters;
  int T, H, E, k;
  int sigmoid, renormalize;
  float routed_scale;
};

// Token t of x -> fp16 image x * 2^(14 - E), E the exponent of its largest magnitude, and 2^(E - 14):
// the largest value lands in [2^14, 2^15); a bf16 or fp16 value keeps all its bits down to 2^-29 of
// the row's largest, and below that errs by at most 2^-40 of it. A NaN or Inf stays one.
template <class X>
__device__ void moe_convert_token(const X* x, __half* xs, float* x_scale, int t, int H,
                                  uint32_t* part) {
  const X* row = x + static_cast<int64_t>(t) * H;
  uint32_t am = 0;
  for (int c = threadIdx.x; c < H / 8; c += kMoeThreads) {
    float v[8];
    load8(row + 8 * c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) am = max(am, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  }
  am = __reduce_max_sync(0xFFFFFFFFu, am);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = am;
  __syncthreads();
  am = 0;
#pragma unroll
  for (int i = 0; i < kMoeWarps; ++i) am = max(am, part[i]);
  const int E = am >= 0x7F800000u ? 14 : max(-100, static_cast<int>(am >> 23) - 127);
  const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - E) << 23);
  for (int c = threadIdx.x; c < H / 8; c += kMoeThreads) {
    float v[8];
    load8(row + 8 * c, v);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(v[2 * j] * up, v[2 * j + 1] * up);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(xs + static_cast<int64_t>(t) * H + moe_perm(8 * c)) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (threadIdx.x == 0) x_scale[t] = __uint_as_float(static_cast<uint32_t>(127 + E - 14) << 23);
}

// One CTA per token, where the caller brings ids and weights.
template <class X>
__global__ void __launch_bounds__(kMoeThreads) moe_prepare_kernel(const X* x, __half* xs,
                                                                 float* x_scale,
                                                                 uint32_t* counters, int H) {
  __shared__ uint32_t part[kMoeWarps];
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (blockIdx.x == 0 && threadIdx.x < kMoeCounters) counters[threadIdx.x] = 0;
  moe_convert_token(x, xs, x_scale, blockIdx.x, H, part);
}

// max (kMax) or sum over the CTA's threads, the same value in all of them, in a fixed order
template <bool kMax>
__device__ __forceinline__ double block_reduce(double v, double* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double u = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = kMax ? fmax(v, u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < kMoeWarps; ++i) v = kMax ? fmax(v, part[i]) : v + part[i];
  return v;
}

// Router: a cluster of eight CTAs per TB tokens; CTA r takes experts r, r + 8, ..., one per warp at
// a time, for all TB tokens; the logits of token i of the group go to CTA i's shared memory, which
// selects for it. Two logits may be arbitrarily close, so they are kept in 64 bits: eight products
// are summed in fp32 and added to a double, an error near 1e-8 of the logits' spread. Bound by the
// latency of one pass over the router weights.
template <class X, class W, int TB>
__global__ void __launch_bounds__(kMoeThreads) moe_route_kernel(const MoeRouteParams p) {
  extern __shared__ double sh[];  // scores [E] (logits of this CTA's token), keys [E]
  __shared__ double part[kMoeWarps];
  __shared__ uint32_t upart[kMoeWarps];
  __shared__ double sel[kMoeMaxTopK];
  const uint32_t rank = cluster_ctarank();
  const int t0 = blockIdx.x / kRouteCluster * TB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const X* x = static_cast<const X*>(p.x);
  const W* wr = static_cast<const W*>(p.router);
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (blockIdx.x == 0 && threadIdx.x < kMoeCounters) p.counters[threadIdx.x] = 0;
  cluster_sync_all();  // every CTA of the cluster runs: its shared memory may be written
  const int pieces = p.H / 8;
  for (int e = rank + kRouteCluster * warp; e < p.E; e += kRouteCluster * kMoeWarps) {
    double acc[TB] = {};
    const W* row = wr + static_cast<int64_t>(e) * p.H;
#pragma unroll 4
    for (int c = lane; c < pieces; c += 32) {
      float w[8];
      load8(row + 8 * c, w);
#pragma unroll
      for (int i = 0; i < TB; ++i) {
        if (t0 + i < p.T) {
          float v[8], s = 0.0f;
          load8(x + static_cast<int64_t>(t0 + i) * p.H + 8 * c, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) s = fmaf(w[j], v[j], s);
          acc[i] += static_cast<double>(s);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < TB; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], o);
      if (lane == 0) {
        const uint32_t at = mapa_shared(smem_u32(&sh[e]), i);
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(acc[i]) : "memory");
      }
    }
  }
  // the fp16 image of token i by CTA 7 - i, while the others may still multiply
  const int mine = kRouteCluster - 1 - static_cast<int>(rank);
  if (mine < TB && t0 + mine < p.T) moe_convert_token(x, p.xs, p.x_scale, t0 + mine, p.H, upart);
  cluster_sync_all();
  const int t = t0 + static_cast<int>(rank);
  if (static_cast<int>(rank) >= TB || t >= p.T) return;
  double* logit = sh;
  double* key = sh + p.E;
  double m = -INFINITY;
  for (int e = threadIdx.x; e < p.E; e += kMoeThreads) m = fmax(m, logit[e]);
  double z = 1.0;
  if (!p.sigmoid) {
    m = block_reduce<true>(m, part);
    z = 0.0;
    for (int e = threadIdx.x; e < p.E; e += kMoeThreads) z += exp(logit[e] - m);
    z = block_reduce<false>(z, part);
  }
  // score in place of the logit; the key ranks: the logit itself (softmax without bias: the same
  // order, nothing rounds), else score + bias; a NaN ranks last
  for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
    const double l = logit[e];
    const double s = p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m) / z;
    const double v = p.bias != nullptr ? s + static_cast<double>(p.bias[e]) : l;
    logit[e] = s;
    key[e] = v == v ? v : -INFINITY;
  }
  __syncthreads();
  // rank of an expert: how many stand before it (ties to the lowest index); ranks are distinct
  for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
    const double v = key[e];
    int r = 0;
    for (int j = 0; j < p.E; ++j) {
      const double u = key[j];
      r += (u > v || (u == v && j < e)) ? 1 : 0;
    }
    if (r < p.k) {
      p.ids[t * p.k + r] = e;
      sel[r] = logit[e];
    }
  }
  __syncthreads();
  if (threadIdx.x < p.k) {
    double sum = 1.0;
    if (p.renormalize) {
      sum = 0.0;
      for (int r = 0; r < p.k; ++r) sum += sel[r];
    }
    p.weights[t * p.k + threadIdx.x] =
        static_cast<float>(sel[threadIdx.x] / sum * static_cast<double>(p.routed_scale));
  }
}

// ---------------------------------------------------------------------------------- kernel 2

struct MoeExpertsParams {
  const uint8_t* w13;        // (E, 2 I, H / 2): gate rows, then up rows
  const uint8_t* s13;        // (E, 2 I, H / 16)
  const float* ts13;         // (E,)
  const uint8_t* w2;         // (E, H, I / 2)
  const uint8_t* s2;         // (E, H, I / 16)
  const float* ts2;
  const int* ids;
  const float* weights;
  const __half* xs;
  const float* x_scale;
  __nv_bfloat16* h;          // (T k, I), permuted
  void* y;                   // (T, H)
  uint32_t* counters;
  int T, H, I, E, k;
  int out_dtype;
  uint32_t* err;
};

__device__ __forceinline__ uint32_t cvt_e2m1x2_f16x2(uint32_t byte) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(r) : "r"(byte));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e4m3x2_f16x2(uint32_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(pair)));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t byte_perm(uint32_t a, uint32_t b, uint32_t s) {
  return __byte_perm(a, b, s);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Streaming load of 16 bytes of weights (read once: not kept in L1).
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// Loads of data written earlier in this grid (h): not through the read-only path.
__device__ __forceinline__ uint4 ld_cg(const void* p) {
  uint4 v;
  asm volatile("ld.global.cg.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_acquire_gpu(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// 8 codes -> four f16x2 of code * scale (adjacent elements), scale in both halves.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t scale, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = mul_f16x2(cvt_e2m1x2_f16x2((w >> (8 * i)) & 0xFFu), scale);
}
// 8 codes -> four bf16x2 of code * scale * 2^-8, element pairs (i, i + 4). The code's three
// magnitude bits sit as bf16 exponent and mantissa bits 8..6 = the value * 2^-126 (subnormals
// included); the scale comes times 2^118.
__device__ __forceinline__ void codes_bf16(uint32_t w, uint32_t scale, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t sg = w << (12 - 4 * i);
    const uint32_t mag = (i < 2 ? w << (6 - 4 * i) : w >> (4 * i - 6)) & 0x01C001C0u;
    o[i] = mul_bf16x2((sg & 0x80008000u) | mag, scale);
  }
}
// Two E4M3 scales (low byte first) times 2^118 as bf16, each in both halves of a word.
__device__ __forceinline__ void scales_bf16(uint32_t pair, uint32_t& s0, uint32_t& s1) {
  const uint32_t h = cvt_e4m3x2_f16x2(pair);
  const __half2 hh = *reinterpret_cast<const __half2*>(&h);
  const float up = __uint_as_float((127u + 118u) << 23);
  const __nv_bfloat162 b =
      __floats2bfloat162_rn(__low2float(hh) * up, __high2float(hh) * up);  // exact (4 bits)
  const uint32_t w = *reinterpret_cast<const uint32_t*>(&b);
  s0 = byte_perm(w, w, 0x1010);
  s1 = byte_perm(w, w, 0x3232);
}

struct MoePlan {
  int cnt[kMoeMaxExperts];           // pairs of an expert
  uint16_t off[kMoeMaxExperts];      // first pair of an expert in `pairs`
  uint16_t act[kMoeMaxExperts];      // experts with at least one pair, ascending
  uint16_t pairs[kMoeMaxTokens * kMoeMaxTopK];  // pairs t * k + slot, by expert
  float w[kMoeMaxTokens * kMoeMaxTopK];         // weight of a pair
  uint8_t tiles[kMoeMaxExperts];     // by active expert: 8-token tiles with a pair (bit mask)
  int nact;
  uint32_t ticket, flag;
};

// Batch of weight loads of a warp: kUnits units (128 elements of K) of two rows.
constexpr int kMoeUnits = 4;
struct MoeBatch {
  uint4 a[kMoeUnits], b[kMoeUnits];
  uint32_t sa[kMoeUnits], sb[kMoeUnits];
};

template <int MAXT>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_experts_kernel(const MoeExpertsParams p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ MoePlan pl;
  constexpr int TP = 8 * MAXT;
  // dynamic: partial sums of the down phase [warps][16][TP] fp32, then pair of (active expert,
  // token) [nact][TP] int16, -1 where the token does not take the expert
  float* red = reinterpret_cast<float*>(dyn);
  int16_t* pair_of = reinterpret_cast<int16_t*>(dyn + kMoeWarps * 16 * TP * 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;
  const int npairs = p.T * p.k;

  for (int e = tid; e < p.E; e += kMoeThreads) pl.cnt[e] = 0;
  __syncthreads();
  grid_dep_wait();
  if (tid == 0) pl.ticket = atomicAdd(p.counters + kMoeShares, 1u);

  // ---- plan: pairs by expert. A token that names an expert twice keeps the first pair with the
  // sum of the weights; ids outside [0, E) are no pair (-1 quietly, others reported).
  int id[(kMoeMaxTokens * kMoeMaxTopK) / kMoeThreads], pos[(kMoeMaxTokens * kMoeMaxTopK) / kMoeThreads];
#pragma unroll
  for (int i = 0; i < kMoeMaxTokens * kMoeMaxTopK / kMoeThreads; ++i) {
    const int pr = tid + i * kMoeThreads;
    id[i] = -1;
    if (pr < npairs) {
      int e = p.ids[pr];
      if (e < 0 || e >= p.E) {
        if (e != -1) atomicOr(p.err, kErrRange);
        e = -1;
      }
      float w = p.weights[pr];
      const int first = pr / p.k * p.k;
      for (int s = first; s < first + p.k && e >= 0; ++s) {
        if (s == pr || p.ids[s] != e) continue;
        if (s < pr) e = -1;
        else w += p.weights[s];
      }
      if (e >= 0) {
        pos[i] = atomicAdd(&pl.cnt[e], 1);
        pl.w[pr] = w;
      }
      id[i] = e;
    }
  }
  __syncthreads();
  if (warp == 0) {
    int nact = 0, off = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int c = e0 + lane < p.E ? pl.cnt[e0 + lane] : 0;
      const uint32_t has = __ballot_sync(0xFFFFFFFFu, c > 0);
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += u;
      }
      if (c > 0) {
        const int a = nact + __popc(has & ((1u << lane) - 1u));
        pl.act[a] = static_cast<uint16_t>(e0 + lane);
        pl.off[e0 + lane] = static_cast<uint16_t>(off + inc - c);
        pl.tiles[a] = 0;
      }
      nact += __popc(has);
      off += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    if (lane == 0) pl.nact = nact;
  }
  __syncthreads();
  const int nact = pl.nact;
#pragma unroll
  for (int i = 0; i < kMoeMaxTokens * kMoeMaxTopK / kMoeThreads; ++i)
    if (id[i] >= 0) pl.pairs[pl.off[id[i]] + pos[i]] = static_cast<uint16_t>(tid + i * kMoeThreads);
  for (int i = tid; i < nact * TP; i += kMoeThreads) pair_of[i] = -1;
  __syncthreads();
  for (int a = warp; a < nact; a += kMoeWarps) {
    const int e = pl.act[a], n = pl.cnt[e];
    uint32_t mask = 0;
    for (int c = lane; c < n; c += 32) {
      const int pr = pl.pairs[pl.off[e] + c];
      pair_of[a * TP + pr / p.k] = static_cast<int16_t>(pr);
      mask |= 1u << (pr / p.k / 8);
    }
    mask = __reduce_or_sync(0xFFFFFFFFu, mask);
    if (lane == 0) pl.tiles[a] = static_cast<uint8_t>(mask);
  }

  // ---- gate / up: granules of 8 hidden units (rows g: gate, g + 8: up of the MMA) over all of H
  const int gpe = p.I / 8;
  const int64_t granules = static_cast<int64_t>(nact) * gpe;
  const int shares = gridDim.x;
  __syncthreads();
  uint32_t share = pl.ticket;
  while (share < static_cast<uint32_t>(shares)) {
    const int64_t g0 = granules * share / shares, g1 = granules * (share + 1) / shares;
    for (int64_t gi = g0 + warp; gi < g1; gi += kMoeWarps) {
      const int a = static_cast<int>(gi / gpe), gl = static_cast<int>(gi % gpe);
      const int e = pl.act[a], n = pl.cnt[e], off = pl.off[e];
      const int nt = (n + 7) / 8;
      const int64_t row = static_cast<int64_t>(e) * 2 * p.I + 8 * gl + g;
      const uint8_t* ca = p.w13 + row * (p.H / 2) + 16 * q;
      const uint8_t* cb = ca + static_cast<int64_t>(p.I) * (p.H / 2);
      const uint8_t* sa = p.s13 + row * (p.H / 16) + 2 * q;
      const uint8_t* sb = sa + static_cast<int64_t>(p.I) * (p.H / 16);
      const __half* xt[MAXT];
#pragma unroll
      for (int i = 0; i < MAXT; ++i) {
        const int c = 8 * i + g;
        xt[i] = c < n ? p.xs + static_cast<int64_t>(pl.pairs[off + c] / p.k) * p.H + 8 * q : nullptr;
      }
      float acc[MAXT][4] = {};
      const int units = p.H / 128;
      MoeBatch cur, nxt;
      auto fetch = [&](MoeBatch& b, int u0) {
#pragma unroll
        for (int i = 0; i < kMoeUnits; ++i)
          if (u0 + i < units) {
            b.a[i] = ld_stream(ca + (u0 + i) * 64);
            b.b[i] = ld_stream(cb + (u0 + i) * 64);
            b.sa[i] = __ldg(reinterpret_cast<const unsigned short*>(sa + (u0 + i) * 8));
            b.sb[i] = __ldg(reinterpret_cast<const unsigned short*>(sb + (u0 + i) * 8));
          }
      };
      fetch(cur, 0);
      for (int u0 = 0; u0 < units; u0 += kMoeUnits) {
        fetch(nxt, u0 + kMoeUnits);
#pragma unroll
        for (int i = 0; i < kMoeUnits; ++i) {
          if (u0 + i >= units) break;
          const uint32_t ha = cvt_e4m3x2_f16x2(cur.sa[i]), hb = cvt_e4m3x2_f16x2(cur.sb[i]);
          const uint32_t wa[4] = {cur.a[i].x, cur.a[i].y, cur.a[i].z, cur.a[i].w};
          const uint32_t wb[4] = {cur.b[i].x, cur.b[i].y, cur.b[i].z, cur.b[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t sel = j < 2 ? 0x1010 : 0x3232;
            uint32_t ga[4], ua[4];
            codes_f16(wa[j], byte_perm(ha, ha, sel), ga);
            codes_f16(wb[j], byte_perm(hb, hb, sel), ua);
#pragma unroll
            for (int m = 0; m < MAXT; ++m) {
              if (m >= nt) break;
              uint4 xb = make_uint4(0, 0, 0, 0);
              if (xt[m] != nullptr)
                xb = __ldg(reinterpret_cast<const uint4*>(xt[m] + (u0 + i) * 128 + 32 * j));
              mma_f16(acc[m], ga[0], ua[0], ga[1], ua[1], xb.x, xb.y);
              mma_f16(acc[m], ga[2], ua[2], ga[3], ua[3], xb.z, xb.w);
            }
          }
        }
        cur = nxt;
      }
      const float ts13 = p.ts13[e], ts2 = p.ts2[e];
      const int at = moe_perm_h(8 * gl + g);
#pragma unroll
      for (int m = 0; m < MAXT; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 8 * m + 2 * q + c;
          if (col < n) {
            const int pr = pl.pairs[off + col];
            const float s = p.x_scale[pr / p.k] * ts13;
            const float gate = acc[m][c] * s, up = acc[m][2 + c] * s;
            const float hv = silu_rn(gate) * up * (pl.w[pr] * ts2);
            p.h[static_cast<int64_t>(pr) * p.I + at] = __float2bfloat16_rn(hv);
          }
        }
    }
    __syncthreads();  // the share's hidden values are written (and the ticket is read)
    if (tid == 0) {
      __threadfence();
      atomicAdd(p.counters + kMoeDone, 1u);
      pl.ticket = atomicAdd(p.counters + kMoeShares, 1u);
    }
    __syncthreads();
    share = pl.ticket;
  }

  // ---- down: tasks of 16 output rows over all active experts and all of I, units (expert,
  // 128-block) dealt to the warps in turn; columns are the tokens, so one accumulator collects
  // every expert's part
  const int tasks = p.H / 16, upe = p.I / 128, units = nact * upe;
  const int per_warp = units > warp ? (units - warp + kMoeWarps - 1) / kMoeWarps : 0;
  bool ready = false;
  while (true) {
    __syncthreads();
    if (tid == 0) pl.ticket = atomicAdd(p.counters + kMoeDown, 1u);
    __syncthreads();
    const uint32_t task = pl.ticket;
    if (task >= static_cast<uint32_t>(tasks)) break;
    const int64_t row = 16 * static_cast<int64_t>(task) + g;
    MoeBatch cur, nxt;
    auto fetch = [&](MoeBatch& b, int v0) {  // v0: number of the unit within this warp's
#pragma unroll
      for (int i = 0; i < kMoeUnits; ++i)
        if (v0 + i < per_warp) {
          const int u = warp + (v0 + i) * kMoeWarps;
          const int a = u / upe, blk = u - a * upe;
          const int64_t r = static_cast<int64_t>(pl.act[a]) * p.H + row;
          const uint8_t* c = p.w2 + r * (p.I / 2) + blk * 64 + 16 * q;
          const uint8_t* s = p.s2 + r * (p.I / 16) + blk * 8 + 2 * q;
          b.a[i] = ld_stream(c);
          b.b[i] = ld_stream(c + static_cast<int64_t>(8) * (p.I / 2));
          b.sa[i] = __ldg(reinterpret_cast<const unsigned short*>(s));
          b.sb[i] = __ldg(reinterpret_cast<const unsigned short*>(s + static_cast<int64_t>(8) * (p.I / 16)));
        }
    };
    fetch(cur, 0);
    if (!ready) {
      // all hidden values (bounded: every share is held by a running CTA)
      if (tid == 0) {
        uint32_t ok = 1;
        const long long c0 = clock64();
        while (ld_acquire_gpu(p.counters + kMoeDone) < static_cast<uint32_t>(shares)) {
          if (static_cast<unsigned long long>(clock64() - c0) > kWaitLimitCycles) {
            atomicOr(p.err, kErrWaitOperand);
            ok = 0;
            break;
          }
        }
        pl.flag = ok;
      }
      __syncthreads();
      if (pl.flag == 0) return;
      ready = true;
    }
    float acc[MAXT][4] = {};
    for (int v0 = 0; v0 < per_warp; v0 += kMoeUnits) {
      fetch(nxt, v0 + kMoeUnits);
#pragma unroll
      for (int i = 0; i < kMoeUnits; ++i) {
        if (v0 + i >= per_warp) break;
        const int u = warp + (v0 + i) * kMoeWarps;
        const int a = u / upe, blk = u - a * upe;
        const uint32_t tiles = pl.tiles[a];
        uint32_t s00, s01, s10, s11;
        scales_bf16(cur.sa[i], s00, s01);
        scales_bf16(cur.sb[i], s10, s11);
        const uint32_t wa[4] = {cur.a[i].x, cur.a[i].y, cur.a[i].z, cur.a[i].w};
        const uint32_t wb[4] = {cur.b[i].x, cur.b[i].y, cur.b[i].z, cur.b[i].w};
        const __nv_bfloat16* ht[MAXT];
#pragma unroll
        for (int m = 0; m < MAXT; ++m) {
          const int pr = pair_of[a * TP + 8 * m + g];
          ht[m] = pr >= 0 ? p.h + static_cast<int64_t>(pr) * p.I + blk * 128 + 8 * q : nullptr;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t ra[4], rb[4];
          codes_bf16(wa[j], j < 2 ? s00 : s01, ra);
          codes_bf16(wb[j], j < 2 ? s10 : s11, rb);
#pragma unroll
          for (int m = 0; m < MAXT; ++m) {
            if (MAXT > 1 && !((tiles >> m) & 1u)) continue;
            uint4 hb = make_uint4(0, 0, 0, 0);
            if (ht[m] != nullptr) hb = ld_cg(ht[m] + 32 * j);
            mma_bf16(acc[m], ra[0], rb[0], ra[1], rb[1], hb.x, hb.y);
            mma_bf16(acc[m], ra[2], rb[2], ra[3], rb[3], hb.z, hb.w);
          }
        }
      }
      cur = nxt;
    }
#pragma unroll
    for (int m = 0; m < MAXT; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        red[(warp * 16 + g + 8 * (c >> 1)) * TP + 8 * m + 2 * q + (c & 1)] = acc[m][c];
    __syncthreads();
    for (int i = tid; i < 16 * p.T; i += kMoeThreads) {
      const int t = i / 16, r = i % 16;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kMoeWarps; ++w) s += red[(w * 16 + r) * TP + t];
      store_out(p.y, static_cast<int64_t>(t) * p.H + 16 * task + r, s * 256.0f, p.out_dtype);
    }
  }
}

}  // namespace bd
