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

// Counters in the workspace, zeroed by the first kernel: tickets and finished tasks per phase.
enum : int {
  kMoeGateUp = 0,
  kMoeGateUpDone = 1,
  kMoeDown = 2,
  kMoeDownDone = 3,
  kMoeCombine = 4,
  kMoeCounters = 5
};

// Position of element k of a row in the scratch images of x and h. A thread of an MMA lane quad q
// takes elements 32 q .. 32 q + 31 of a 128-block (one 16-byte piece of the weights' codes), in four
// loads of 8: load j of the quad is 64 contiguous bytes when (q, j) are exchanged.
__host__ __device__ __forceinline__ int moe_perm(int k) {
  const int r = k & 127;
  return (k & ~127) + ((r >> 3) & 3) * 32 + (r >> 5) * 8 + (r & 7);
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
  uint32_t* hmax;
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
                                                                 uint32_t* counters,
                                                                 uint32_t* hmax, int H, int k) {
  __shared__ uint32_t part[kMoeWarps];
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (blockIdx.x == 0 && threadIdx.x < kMoeCounters) counters[threadIdx.x] = 0;
  if (threadIdx.x < k) hmax[blockIdx.x * k + threadIdx.x] = 0;
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
    p.hmax[t * p.k + threadIdx.x] = 0;
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
  float* h;                  // (T k, I) hidden values times weight and down scale
  uint32_t* hmax;            // (T k,) bits of the largest |h| of a pair, zeroed by kernel 1
  float* part;               // (slices, T k, H) partial sums; part_rows rows in all
  void* y;                   // (T, H)
  uint32_t* counters;
  int T, H, I, E, k;
  int part_rows;
  int out_dtype, vec_out;
  uint32_t* err;
};

// 8 codes (four bytes) -> four f16x2.
__device__ __forceinline__ void cvt_e2m1x8_f16(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
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
  cvt_e2m1x8_f16(w, o);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = mul_f16x2(o[i], scale);
}
struct MoePlan {
  int cnt[kMoeMaxExperts];           // pairs of an expert
  uint16_t off[kMoeMaxExperts];      // first pair of an expert in `pairs`
  uint16_t act[kMoeMaxExperts];      // experts with at least one pair, ascending
  uint16_t pairs[kMoeMaxTokens * kMoeMaxTopK];  // pairs t * k + slot, by expert
  float w[kMoeMaxTokens * kMoeMaxTopK];         // weight of a pair
  uint8_t used[kMoeMaxTokens * kMoeMaxTopK];    // the pair counts
  int nact;
  uint32_t ticket, flag;
  uint32_t hmax[32];
};

// Pairs by expert. A token that names an expert twice keeps the first pair with the sum of the
// weights; ids outside [0, E) are no pair (-1 quietly, others reported). Ends with a barrier.
__device__ void moe_plan(const MoeExpertsParams& p, MoePlan& pl) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int npairs = p.T * p.k;
  constexpr int kPer = kMoeMaxTokens * kMoeMaxTopK / kMoeThreads;
  int id[kPer], pos[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int pr = tid + i * kMoeThreads;
    id[i] = -1;
    pos[i] = 0;
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
      pl.used[pr] = e >= 0;
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
        pl.act[nact + __popc(has & ((1u << lane) - 1u))] = static_cast<uint16_t>(e0 + lane);
        pl.off[e0 + lane] = static_cast<uint16_t>(off + inc - c);
      }
      nact += __popc(has);
      off += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    if (lane == 0) pl.nact = nact;
  }
  __syncthreads();
  // the place of a pair within its expert's list is the order of arrival: it picks an MMA
  // column, not a value
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (id[i] >= 0) pl.pairs[pl.off[id[i]] + pos[i]] = static_cast<uint16_t>(tid + i * kMoeThreads);
  __syncthreads();
}

// tid 0: until *counter >= target (bounded); the others take the answer from pl.flag after a
// barrier. The writes counted before are visible to the CTA afterwards.
__device__ __forceinline__ bool moe_wait(const uint32_t* counter, uint32_t target, MoePlan& pl,
                                         uint32_t* err) {
  if (threadIdx.x == 0) {
    uint32_t ok = 1;
    const long long c0 = clock64();
    while (ld_acquire_gpu(counter) < target) {
      if (static_cast<unsigned long long>(clock64() - c0) > kWaitLimitCycles) {
        atomicOr(err, kErrWaitOperand);
        ok = 0;
        break;
      }
    }
    pl.flag = ok;
  }
  __syncthreads();
  return pl.flag != 0;
}

// Exponent that takes a row whose largest magnitude has these bits to [2^14, 2^15) (fp16): the row
// times 2^(14 - E).
__device__ __forceinline__ int moe_row_exp(uint32_t amax_bits) {
  return amax_bits >= 0x7F800000u ? 14 : max(-100, static_cast<int>(amax_bits >> 23) - 127);
}
__device__ __forceinline__ float pow2f(int e) {
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// Weights of one unit (128 elements of K) of a warp's 16 MB rows: per MMA row block the 16 code
// bytes and two scale bytes of this lane in rows g and g + 8.
template <int MB>
struct MoeUnit {
  uint4 a[MB], b[MB];
  uint32_t sa[MB], sb[MB];
};
struct MoeRows {
  const uint8_t *codes, *scales;  // this lane's place in row g of the warp's first row block
  int64_t block, second;          // bytes of codes from row block to row block, from row g to g + 8
};
template <int MB>
__device__ __forceinline__ void moe_fetch(MoeUnit<MB>& w, const MoeRows& r, int u) {
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const uint8_t* c = r.codes + m * r.block + u * 64;
    const uint8_t* s = r.scales + (m * r.block >> 3) + u * 8;
    w.a[m] = ld_stream(c);
    w.b[m] = ld_stream(c + r.second);
    w.sa[m] = __ldg(reinterpret_cast<const unsigned short*>(s));
    w.sb[m] = __ldg(reinterpret_cast<const unsigned short*>(s + (r.second >> 3)));
  }
}

constexpr int kMoeTiles = 4;                // token tiles (8 columns each) per pass over the weights
constexpr int kMoeBBytes = 72 * 1024;       // staged activations
constexpr int kMoePad = 64;                 // bytes between token rows: conflict-free 16-byte reads

// One unit against nt staged token tiles: tok is this lane's place in the staged block (token row g
// of tile 0, 16 bytes per MMA pair), `tile` bytes on to the next tile.
template <int MB, int NT>
__device__ __forceinline__ void moe_unit(float (&acc)[MB][kMoeTiles][4], const MoeUnit<MB>& w,
                                         uint32_t tok, uint32_t tile) {
  uint32_t ha[MB], hb[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    ha[m] = cvt_e4m3x2_f16x2(w.sa[m]);
    hb[m] = cvt_e4m3x2_f16x2(w.sb[m]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 xb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(xb[t].x), "=r"(xb[t].y), "=r"(xb[t].z), "=r"(xb[t].w)
                   : "r"(tok + t * tile + 64 * j));
    const uint32_t sel = j < 2 ? 0x1010 : 0x3232;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const uint32_t wa = j == 0 ? w.a[m].x : j == 1 ? w.a[m].y : j == 2 ? w.a[m].z : w.a[m].w;
      const uint32_t wb = j == 0 ? w.b[m].x : j == 1 ? w.b[m].y : j == 2 ? w.b[m].z : w.b[m].w;
      uint32_t fa[4], fb[4];
      codes_f16(wa, byte_perm(ha[m], ha[m], sel), fa);
      codes_f16(wb, byte_perm(hb[m], hb[m], sel), fb);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        mma_f16(acc[m][t], fa[0], fb[0], fa[1], fb[1], xb[t].x, xb[t].y);
        mma_f16(acc[m][t], fa[2], fb[2], fa[3], fb[3], xb[t].z, xb[t].w);
      }
    }
  }
}

// Units [u0, u1) of a warp's rows against the staged block that begins with unit u0; w holds the
// weights of u0 and ends with those of u1 (when u1 < end).
template <int MB, int NT>
__device__ __forceinline__ void moe_run(float (&acc)[MB][kMoeTiles][4], MoeUnit<MB>& w,
                                        const MoeRows& rows, int u0, int u1, int end,
                                        uint32_t tok, uint32_t tile) {
  MoeUnit<MB> nxt;
  int u = u0;
#pragma unroll 1
  for (; u + 2 <= u1; u += 2, tok += 512) {
    moe_fetch(nxt, rows, u + 1);
    moe_unit<MB, NT>(acc, w, tok, tile);
    if (u + 2 < end) moe_fetch(w, rows, u + 2);
    moe_unit<MB, NT>(acc, nxt, tok + 256, tile);
  }
  if (u < u1) {
    if (u + 1 < end) moe_fetch(nxt, rows, u + 1);
    moe_unit<MB, NT>(acc, w, tok, tile);
    w = nxt;
  }
}
template <int MB>
__device__ __forceinline__ void moe_run(float (&acc)[MB][kMoeTiles][4], MoeUnit<MB>& w,
                                        const MoeRows& rows, int u0, int u1, int end,
                                        uint32_t tok, uint32_t tile, int nt) {
  if (nt == 1) moe_run<MB, 1>(acc, w, rows, u0, u1, end, tok, tile);
  else if (nt == 2) moe_run<MB, 2>(acc, w, rows, u0, u1, end, tok, tile);
  else if (nt == 3) moe_run<MB, 3>(acc, w, rows, u0, u1, end, tok, tile);
  else moe_run<MB, 4>(acc, w, rows, u0, u1, end, tok, tile);
}

// The experts' kernel. Tasks of 8 warps x 16 MB weight rows of one expert, all of the expert's tokens
// (in passes of 32 where more take it), K streamed: weights from global memory to registers one unit
// ahead, activations staged in shared memory for all eight warps, as much of K at a time as fits.
//   gate / up: 64 MB hidden units (MMA row g: gate, g + 8: up of one unit, so one thread holds both
//              values of the same token); h = silu(gate) up w ts in fp32, and its row maximum;
//   down:      128 MB output rows of one expert and a slice of I; h staged as fp16 times the power of
//              two that brings its row's maximum to [2^14, 2^15); partial sums per (slice, pair);
//   combine:   y = the partial sums of a token's pairs in slot order.
// Each phase's tasks wait for the phase before (see the ticket argument at the top).
template <int MB>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_experts_kernel(const MoeExpertsParams p) {
  extern __shared__ __align__(16) uint8_t stage[];
  __shared__ MoePlan pl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;

  for (int e = tid; e < p.E; e += kMoeThreads) pl.cnt[e] = 0;
  __syncthreads();
  grid_dep_wait();
  if (tid == 0) pl.ticket = atomicAdd(p.counters + kMoeGateUp, 1u);
  moe_plan(p, pl);
  const int nact = pl.nact;

  const int blocks1 = p.I / (64 * MB);
  const uint32_t total1 = static_cast<uint32_t>(nact) * blocks1;
  const int blocks2 = (p.H + 128 * MB - 1) / (128 * MB);
  const int units2 = p.I / 128;
  // slices of I per down task: while the tasks do not fill the grid and the partials fit
  int slices = 1;
  while (nact * blocks2 * slices < static_cast<int>(gridDim.x) &&
         2 * slices * p.T * p.k <= p.part_rows && units2 >= 4 * slices)
    slices *= 2;
  const uint32_t total2 = static_cast<uint32_t>(nact) * blocks2 * slices;

  // tokens [c0, c0 + n) of an expert: geometry of the staged block
  auto chunk_units = [](int n8) { return min((kMoeBBytes / n8 - kMoePad) / 256, 1 << 20); };
  const uint32_t stage_u = smem_u32(stage);

  // ------------------------------------------------------------------------------ gate / up
  while (true) {
    const uint32_t task = pl.ticket;
    if (task >= total1) break;
    const int a = task / blocks1, blk = task % blocks1;
    const int e = pl.act[a], cnt = pl.cnt[e], off = pl.off[e];
    const int i0 = blk * 64 * MB + warp * 8 * MB;  // this warp's first hidden unit
    const int units = p.H / 128;
    MoeRows rows;
    {
      const int64_t row = static_cast<int64_t>(e) * 2 * p.I + i0 + g;
      rows.codes = p.w13 + row * (p.H / 2) + 16 * q;
      rows.scales = p.s13 + row * (p.H / 16) + 2 * q;
      rows.block = static_cast<int64_t>(8) * (p.H / 2);
      rows.second = static_cast<int64_t>(p.I) * (p.H / 2);
    }
    const float ts13 = p.ts13[e], ts2 = p.ts2[e];
    for (int c0 = 0; c0 < cnt; c0 += 8 * kMoeTiles) {
      const int n = min(cnt - c0, 8 * kMoeTiles), nt = (n + 7) / 8;
      const int cu = chunk_units(8 * nt);
      float acc[MB][kMoeTiles][4] = {};
      MoeUnit<MB> cur;
      moe_fetch(cur, rows, 0);
      for (int u0 = 0; u0 < units; u0 += cu) {
        const int uc = min(cu, units - u0);
        const uint32_t pitch = uc * 256 + kMoePad;
        if (u0 > 0) __syncthreads();  // the block staged before is read
        for (int c = warp; c < 8 * nt; c += kMoeWarps) {
          const int4* src = reinterpret_cast<const int4*>(
              c < n ? p.xs + static_cast<int64_t>(pl.pairs[off + c0 + c] / p.k) * p.H + u0 * 128
                    : nullptr);
          for (int i = lane; i < uc * 16; i += 32) {
            const uint32_t dst = stage_u + c * pitch + i * 16;
            if (src != nullptr)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src + i)
                           : "memory");
            else
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(dst), "r"(0) : "memory");
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        moe_run<MB>(acc, cur, rows, u0, u0 + uc, units, stage_u + g * pitch + 16 * q, 8 * pitch, nt);
      }
      if (tid < 32) pl.hmax[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int t = 0; t < kMoeTiles; ++t) {
        if (t >= nt) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 8 * t + 2 * q + c;
          uint32_t hm = 0;
          if (col < n) {
            const int pr = pl.pairs[off + c0 + col];
            const float s = p.x_scale[pr / p.k] * ts13, wt = pl.w[pr] * ts2;
#pragma unroll
            for (int m = 0; m < MB; ++m) {
              const float h = silu_rn(acc[m][t][c] * s) * (acc[m][t][2 + c] * s) * wt;
              p.h[static_cast<int64_t>(pr) * p.I + i0 + 8 * m + g] = h;
              hm = max(hm, __float_as_uint(h) & 0x7FFFFFFFu);
            }
          }
          hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, 4));
          hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, 8));
          hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, 16));
          if (g == 0 && col < n) atomicMax(&pl.hmax[col], hm);
        }
      }
      __syncthreads();
      if (tid < n) atomicMax(p.hmax + pl.pairs[off + c0 + tid], pl.hmax[tid]);
    }
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      atomicAdd(p.counters + kMoeGateUpDone, 1u);
      pl.ticket = atomicAdd(p.counters + kMoeGateUp, 1u);
    }
    __syncthreads();
  }

  // ---------------------------------------------------------------------------------- down
  bool ready = false;
  while (true) {
    __syncthreads();
    if (tid == 0) pl.ticket = atomicAdd(p.counters + kMoeDown, 1u);
    __syncthreads();
    const uint32_t task = pl.ticket;
    if (task >= total2) break;
    const int z = task % slices, ab = task / slices;
    const int a = ab / blocks2, blk = ab % blocks2;
    const int e = pl.act[a], cnt = pl.cnt[e], off = pl.off[e];
    const int r0 = blk * 128 * MB + warp * 16 * MB;  // this warp's first output row
    const bool active = r0 < p.H;                   // H % 128 == 0: whole warps
    const int ub = static_cast<int>(static_cast<int64_t>(units2) * z / slices);
    const int ue = static_cast<int>(static_cast<int64_t>(units2) * (z + 1) / slices);
    MoeRows rows;
    {
      const int64_t row = static_cast<int64_t>(e) * p.H + (active ? r0 : 0) + g;
      rows.codes = p.w2 + row * (p.I / 2) + 16 * q;
      rows.scales = p.s2 + row * (p.I / 16) + 2 * q;
      rows.block = static_cast<int64_t>(16) * (p.I / 2);
      rows.second = static_cast<int64_t>(8) * (p.I / 2);
    }
    for (int c0 = 0; c0 < cnt; c0 += 8 * kMoeTiles) {
      const int n = min(cnt - c0, 8 * kMoeTiles), nt = (n + 7) / 8;
      const int cu = chunk_units(8 * nt);
      float acc[MB][kMoeTiles][4] = {};
      MoeUnit<MB> cur;
      moe_fetch(cur, rows, ub);
      if (!ready) {
        if (!moe_wait(p.counters + kMoeGateUpDone, total1, pl, p.err)) return;
        ready = true;
      }
      for (int u0 = ub; u0 < ue; u0 += cu) {
        const int uc = min(cu, ue - u0);
        const uint32_t pitch = uc * 256 + kMoePad;
        __syncthreads();
        for (int c = warp; c < 8 * nt; c += kMoeWarps) {
          const int pr = c < n ? pl.pairs[off + c0 + c] : -1;
          const float* src = pr >= 0 ? p.h + static_cast<int64_t>(pr) * p.I + u0 * 128 : nullptr;
          const float up = pr >= 0 ? pow2f(14 - moe_row_exp(__ldcg(p.hmax + pr))) : 0.0f;
          for (int i = lane; i < uc * 16; i += 32) {
            // piece i of the permuted row: elements 32 q + 8 j .. + 7 of block i / 16
            uint32_t w[4] = {0, 0, 0, 0};
            if (src != nullptr) {
              const float* s = src + (i >> 4) * 128 + 32 * (i & 3) + 8 * ((i >> 2) & 3);
              const uint4 lo = ld_cg(s), hi = ld_cg(s + 4);
              const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const __half2 hh = __floats2half2_rn(__uint_as_float(v[2 * j]) * up,
                                                     __uint_as_float(v[2 * j + 1]) * up);
                w[j] = *reinterpret_cast<const uint32_t*>(&hh);
              }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage_u + c * pitch + i * 16),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
        }
        __syncthreads();
        if (active)
          moe_run<MB>(acc, cur, rows, u0, u0 + uc, ue, stage_u + g * pitch + 16 * q, 8 * pitch, nt);
      }
      if (active) {
#pragma unroll
        for (int t = 0; t < kMoeTiles; ++t) {
          if (t >= nt) break;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int col = 8 * t + 2 * q + c;
            if (col < n) {
              const int pr = pl.pairs[off + c0 + col];
              const float back = pow2f(moe_row_exp(__ldcg(p.hmax + pr)) - 14);
              float* dst = p.part + (static_cast<int64_t>(z) * p.T * p.k + pr) * p.H + r0 + g;
#pragma unroll
              for (int m = 0; m < MB; ++m) {
                dst[16 * m] = acc[m][t][c] * back;
                dst[16 * m + 8] = acc[m][t][2 + c] * back;
              }
            }
          }
        }
      }
    }
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      atomicAdd(p.counters + kMoeDownDone, 1u);
    }
  }

  // -------------------------------------------------------------------------------- combine
  const int cols = 4 * kMoeThreads;  // outputs per task
  const int blocks3 = (p.H + cols - 1) / cols;
  ready = false;
  while (true) {
    __syncthreads();
    if (tid == 0) pl.ticket = atomicAdd(p.counters + kMoeCombine, 1u);
    __syncthreads();
    const uint32_t task = pl.ticket;
    if (task >= static_cast<uint32_t>(p.T * blocks3)) break;
    if (!ready) {
      if (!moe_wait(p.counters + kMoeDownDone, total2, pl, p.err)) return;
      ready = true;
    }
    const int t = task / blocks3, h0 = (task % blocks3) * cols + 4 * tid;
    if (h0 >= p.H) continue;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < p.k; ++s) {
      const int pr = t * p.k + s;
      if (!pl.used[pr]) continue;
      for (int z = 0; z < slices; ++z) {
        const uint4 v =
            ld_cg(p.part + (static_cast<int64_t>(z) * p.T * p.k + pr) * p.H + h0);
        o[0] += __uint_as_float(v.x);
        o[1] += __uint_as_float(v.y);
        o[2] += __uint_as_float(v.z);
        o[3] += __uint_as_float(v.w);
      }
    }
    store_row<4>(p.y, static_cast<int64_t>(t) * p.H + h0, o, p.out_dtype, p.vec_out);
  }
}

}  // namespace bd
