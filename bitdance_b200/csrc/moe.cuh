// moe.cuh -- a mixture-of-experts layer for a few tokens (T <= 64) in two kernels, expert weights
// in NVFP4 as bd_quantize_b_nvfp4 writes them (natural codes and scales, nothing packed):
//
//   logits = x Wr^T;  s = softmax or sigmoid(logits);  top-k by s (+ bias);  w = s (renormalised)
//   y_t = sum over the chosen experts e of w_e * Wd_e (silu(Wg_e x_t) * (Wu_e x_t))
//
// A few tokens read far more weights than they compute with: the time is that of streaming the touched
// experts' 4-bit weights once. So no thread touches a weight: codes and scales go by TMA and
// cp.async to shared memory and from there to tcgen05.mma kind::mxf4nvf4 as they are. What that MMA
// wants besides is a second operand in 4 bits, and it has columns to spare: a token becomes eight
// columns, six of them digits of its values. With s = 2^e the scale of a 16-block (amax <= 4 s),
//   x = s (d_0 + d_1 / 8 + ... + d_5 / 8^5) + r,   d_p = E2M1 round of what is left, |r| <= s 2^-16.
// All six digits carry the block's scale s, an E4M3 power of two; a digit's factor 8^-p is common to its
// column, so it is applied to the column's finished sum. The product is then one with x to 2^-17 of the
// block's largest value, or to 2^-34 of the row's where E4M3's smallest scale is larger than the block
// wants: activations of 16 bits against 4-bit weights (W4A16) on the FP4 tensor cores without unpacking
// a weight. (Unpacking them into fp16 fragments for mma.sync took 140 to 175 instructions per 2048
// weights and ran at 40 % of the memory rate.)
//
// Kernel 1 (moe_route_kernel, or moe_prepare_kernel where the caller brings the routing): router
// products, selection, digits of x, counters to zero.
// Kernel 2 (moe_experts_kernel): gate / up, digits of the hidden values, down and combine phases in
// one grid. Work is handed out by tickets (atomic counters) in the order of the experts, and a task
// waits only for the tasks of its own expert. All gate / up tickets go before the first down ticket,
// and no gate / up task waits for anything: whatever a CTA waits for is held by a CTA that already
// runs, so the waits end without any guarantee that the whole grid is resident.
#pragma once
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "epilogue.cuh"
#include "sm100.cuh"

namespace bd {

constexpr int kMoeMaxTokens = 64, kMoeMaxExperts = 512, kMoeMaxTopK = 16;
constexpr int kMoeThreads = 512, kMoeWarps = kMoeThreads / 32;
constexpr int kRouteCluster = 8;

// Counters in the workspace, zeroed by the first kernel: tickets and finished tasks, then per touched
// expert its finished gate / up tasks [E] and digit tasks [E].
enum : int {
  kMoeGateUp = 0,
  kMoeDigits,
  kMoeDigitsDone,
  kMoeDown,
  kMoeDownDone,
  kMoeCounters
};
__host__ __device__ constexpr int moe_counters(int E) { return kMoeCounters + 2 * E; }

// Digits of a row of K activations: per 256 elements the 8 x 128 bytes of codes (row p: digit p; rows
// 6 and 7 are zero), 128B-swizzled as the MMA's operand tile, then 8 x 4 words of scales (the same
// for every row).
constexpr int kMoeDigitRows = 8, kMoeDigitCount = 6;
constexpr int kMoeChunkCodes = 1024;
constexpr int kMoeChunk = kMoeChunkCodes + 128;
__host__ __device__ __forceinline__ int64_t moe_image_row(int K) {
  return static_cast<int64_t>((K + 255) / 256) * kMoeChunk;
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
  uint8_t* xs;             // digits of x
  float* x_scale;          // (T,) row factors
  uint32_t* hmax;          // (T, k) zeroed here
  uint32_t* counters;
  int T, H, E, k;
  int sigmoid, renormalize;
  float routed_scale;
};

__device__ __forceinline__ float pow2f(int e) {
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
// Row factor: with 2^E <= amax < 2^(E+1) the row times 2^(9 - E) is below 2^10 = 4 * 2^8, so that its
// largest block's scale is E4M3's 2^8. Returns 9 - E; the factor back is 2^(E - 9), and NaN for a
// row with a NaN or Inf (its digits are finite: the factor carries the NaN into every product). Rows
// below 2^-100 get the factor of 2^-100.
__device__ __forceinline__ int moe_row_shift(uint32_t amax_bits) {
  return 9 - min(127, max(-100, static_cast<int>(amax_bits >> 23) - 127));
}
__device__ __forceinline__ float moe_row_factor(uint32_t amax_bits) {
  return amax_bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u)
                                  : pow2f(-moe_row_shift(amax_bits));
}

// E2M1 codes of (lo, hi), round to nearest, and their values.
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi, float& vlo, float& vhi) {
  uint32_t code, val;
  asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %3, %2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.u32.u8 %0, b;\n\t}"
      : "=r"(code), "=r"(val)
      : "f"(lo), "f"(hi));
  const __half2 h = *reinterpret_cast<const __half2*>(&val);
  vlo = __low2float(h);
  vhi = __high2float(h);
  return code;
}

// Digits of the 16-block `blk` of a row (values v already times the row's 2^shift) into its image.
// Lanes 4 i .. 4 i + 3 hold four consecutive blocks (one scale word); all lanes of a group come
// together. One digit after the other in the code: a warp comes by few times, and the instructions' way
// from memory counts (side by side, 48 tokens 110 us for 108, 7 tokens 90 for 86.5, large experts equal).
__device__ __forceinline__ void moe_digits(float (&v)[16], uint8_t* img, int blk) {
  float a = 0.0f;
#pragma unroll
  for (int j = 0; j < 16; ++j) a = fmaxf(a, fabsf(v[j]));
  const int e = max(-9, min(8, static_cast<int>(__float_as_uint(a) >> 23) - 128));  // amax <= 4 2^e
  const float down = pow2f(-e);
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] *= down;
  uint8_t* chunk = img + static_cast<int64_t>(blk >> 4) * kMoeChunk;
  const int piece = (blk & 15) >> 1;  // 16-byte piece of the 128-byte row; this block is half of it
  const uint32_t group = 0xFu << (threadIdx.x & 28);
  const uint32_t byte = e >= -6 ? static_cast<uint32_t>(e + 7) << 3 : 1u << (e + 9);  // E4M3 2^e
  uint32_t word = byte << (8 * (blk & 3));
  word |= __shfl_xor_sync(group, word, 1);
  word |= __shfl_xor_sync(group, word, 2);
  uint8_t* scales = chunk + kMoeChunkCodes + (blk & 12);  // rows 2 i and 2 i + 1 by lane i of the four
  *reinterpret_cast<uint32_t*>(scales + (blk & 3) * 32) = word;
  *reinterpret_cast<uint32_t*>(scales + (blk & 3) * 32 + 16) = word;
#pragma unroll 1
  for (int p = 0; p < kMoeDigitRows; ++p) {
    uint32_t w[2] = {0, 0};
    if (p < kMoeDigitCount) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float d0, d1;
        w[j >> 2] |= e2m1_pair(v[2 * j], v[2 * j + 1], d0, d1) << (8 * (j & 3));
        v[2 * j] = (v[2 * j] - d0) * 8.0f;
        v[2 * j + 1] = (v[2 * j + 1] - d1) * 8.0f;
      }
    }
    *reinterpret_cast<uint2*>(chunk + p * 128 + ((piece ^ p) << 4) + (blk & 1) * 8) =
        make_uint2(w[0], w[1]);
  }
}

// Digits of token t of x, by one CTA.
template <class X>
__device__ void moe_convert_token(const X* x, uint8_t* xs, float* x_scale, int t, int H,
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
  const float up = pow2f(moe_row_shift(am));
  for (int b = threadIdx.x; b < H / 16; b += kMoeThreads) {  // H / 16 is a multiple of 8
    float v[16];
    load8(row + 16 * b, *reinterpret_cast<float(*)[8]>(v));
    load8(row + 16 * b + 8, *reinterpret_cast<float(*)[8]>(v + 8));
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] *= up;
    moe_digits(v, xs + t * moe_image_row(H), b);
  }
  if (threadIdx.x == 0) x_scale[t] = moe_row_factor(am);
}

// One CTA per token, where the caller brings ids and weights.
template <class X>
__global__ void __launch_bounds__(kMoeThreads)
    moe_prepare_kernel(const X* x, uint8_t* xs, float* x_scale, uint32_t* hmax, uint32_t* counters,
                       int H, int E, int k) {
  __shared__ uint32_t part[kMoeWarps];
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < moe_counters(E); i += kMoeThreads) counters[i] = 0;
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

// A logit in 64 bits, by a warp: a lane's 8-element pieces c, c + step, ... kExact: each product in 64 bits
// too; else in fp32, where a product of two 16-bit numbers is exact unless it leaves fp32's range. some: x
// is not zero throughout.
template <bool kExact, int kUnroll, class X, class W>
__device__ __forceinline__ double route_dot(const W* row, const X* x, int c, int step, int pieces,
                                            bool& some) {
  double sum[4] = {};
  uint32_t bits = 0;
#pragma unroll kUnroll
  for (; c < pieces; c += step) {
    float w[8], v[8];
    load8(row + 8 * c, w);
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(x + 8 * c));
    bits |= q.x | q.y | q.z | q.w;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(reinterpret_cast<const X*>(&q)[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (kExact) sum[j & 3] = fma(static_cast<double>(w[j]), static_cast<double>(v[j]), sum[j & 3]);
      else sum[j & 3] += static_cast<double>(__fmul_rn(w[j], v[j]));
    }
  }
  double all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
  some = __any_sync(0xFFFFFFFFu, bits != 0);
  return all;
}

// Router: a cluster of eight CTAs per token; a CTA takes every eighth expert (every seventh, and the last
// CTA none, where seven CTAs' warps hold all experts at once), a warp per expert and part of K (of eight
// where the experts are few); the partial logits go to CTA 0's shared memory, which adds and selects. The
// last CTA makes the token's digits meanwhile. Two logits may be arbitrarily close, so they are sums in 64
// bits of exact products: of 16-bit routers in fp32, one conversion each (eight products summed in fp32
// first misplaced logits closer than 2^-24 of their terms; the layer of 48 tokens and 128 experts takes 105
// us either way, of 7 tokens, H 4096, 83 for 81, of 64 tokens and 512 experts 144 for 140), again with
// 64-bit products where one may have left fp32's range (a sum that is not finite, or so small that what
// underflowed could count); of fp32 routers in 64 bits (16 tokens, 256 experts, H 4096 89 us for 85). Bound
// by latency: one pass over the router weights is half of it (3 of 5 us for one token and 64 experts), the
// selection's steps the rest. (Two or four tokens per cluster, for fewer passes over the weights: 64
// tokens, 64 experts, H 4096 took the layer 127 us for 118. A share of the token's digits in each CTA took
// longer than one CTA's whole token beside the others' products: 17 for 14 us at seven tokens.)
template <class X, class W, int parts>
__global__ void __launch_bounds__(kMoeThreads) moe_route_kernel(const MoeRouteParams p) {
  extern __shared__ double sh[];  // partial logits [parts][E], then keys [E]
  __shared__ double part[kMoeWarps];
  __shared__ uint32_t upart[kMoeWarps];
  __shared__ double sel[kMoeMaxTopK];
  const int rank = static_cast<int>(cluster_ctarank()), t = blockIdx.x / kRouteCluster;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const X* x = static_cast<const X*>(p.x);
  const W* wr = static_cast<const W*>(p.router);
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < moe_counters(p.E); i += kMoeThreads) p.counters[i] = 0;
  cluster_sync_all();  // every CTA of the cluster runs: its shared memory may be written
  const int pieces = p.H / 8;
  const int ranks = p.E <= (kRouteCluster - 1) * kMoeWarps ? kRouteCluster - 1 : kRouteCluster;
  const int experts = rank < ranks ? (p.E - rank + ranks - 1) / ranks : 0;
  for (int job = warp; job < experts * parts; job += kMoeWarps) {
    const int e = rank + ranks * (job / parts), q = job % parts;
    const W* row = wr + static_cast<int64_t>(e) * p.H;
    const X* xt = x + static_cast<int64_t>(t) * p.H;
    constexpr bool kExact = sizeof(W) == 4;
    bool some;
    double acc = route_dot<kExact, 8>(row, xt, 32 * q + lane, 32 * parts, pieces, some);
    // products of two bf16 numbers may leave fp32's range (of fp16 none does): 2^20 of them below 2^-126 lose
    // 2^-130 in all, nothing beside 2^-60 in 64 bits. (Zero rows pad a batch: they cost no second pass.)
    if constexpr (!kExact && std::is_same_v<X, __nv_bfloat16>) {
      if (some && !(fabs(acc) > 8.7e-19 && fabs(acc) < INFINITY))
        acc = route_dot<true, 1>(row, xt, 32 * q + lane, 32 * parts, pieces, some);
    }
    if (lane == 0) {
      const uint32_t at = mapa_shared(smem_u32(&sh[q * p.E + e]), 0);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(acc) : "memory");
    }
  }
  if (rank == kRouteCluster - 1) moe_convert_token(x, p.xs, p.x_scale, t, p.H, upart);
  cluster_sync_all();
  if (rank != 0) return;
  // Scores and keys. The key ranks: the logit itself (softmax without bias: the same order, nothing
  // rounds), else score + bias; a NaN ranks last. Where the weights are renormalised softmax scores
  // ranked by logit, exp(logit - largest) of the chosen ones is all that is needed (and whether any logit
  // is a NaN: then every score is).
  double* score = sh;
  double* key = sh + parts * p.E;
  const bool lazy = !p.sigmoid && p.bias == nullptr && p.renormalize;
  bool nan = false;
  for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
    double l = score[e];
#pragma unroll
    for (int q = 1; q < parts; ++q) l += sh[q * p.E + e];
    if (parts > 1) score[e] = l;
    key[e] = l == l ? l : -INFINITY;
    nan |= l != l;
  }
  if (!lazy) {  // (every loop gives a thread the same experts)
    double m = 0.0, z = 1.0;
    if (!p.sigmoid) {
      m = -INFINITY;
      for (int e = threadIdx.x; e < p.E; e += kMoeThreads) m = fmax(m, score[e]);
      m = block_reduce<true>(m, part);
      z = 0.0;
      for (int e = threadIdx.x; e < p.E; e += kMoeThreads) z += exp(score[e] - m);
      z = block_reduce<false>(z, part);
    }
    for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
      const double l = score[e];
      const double s = p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m) / z;
      const double v = p.bias != nullptr ? s + static_cast<double>(p.bias[e]) : l;
      score[e] = s;
      key[e] = v == v ? v : -INFINITY;
    }
  }
  nan = __syncthreads_or(nan);
  // rank of an expert: how many stand before it (ties to the lowest index); ranks are distinct.
  // `team` threads (a power of two up to 32) share an expert.
  int team = 32;
  while (team > 1 && team * p.E > kMoeThreads) team >>= 1;
  const int sub = threadIdx.x & (team - 1);
  for (int e0 = 0; e0 < p.E; e0 += kMoeThreads / team) {
    const int e = e0 + threadIdx.x / team;
    int r = 0;
    if (e < p.E) {
      const double v = key[e];
#pragma unroll 8
      for (int j = sub; j < p.E; j += team) {
        const double u = key[j];
        r += (u > v || (u == v && j < e)) ? 1 : 0;
      }
    }
    for (int o = team >> 1; o > 0; o >>= 1) r += __shfl_xor_sync(0xFFFFFFFFu, r, o);
    if (e < p.E && sub == 0 && r < p.k) {
      p.ids[t * p.k + r] = e;
      sel[r] = score[e];
    }
  }
  __syncthreads();
  if (warp == 0) {
    // lazy: sel holds logits, the first the largest (all NaN or -inf: the weights are NaN, as theirs)
    double mine = lane < p.k ? sel[lane] : 0.0, sum = 1.0;
    if (lazy && lane < p.k) mine = exp(mine - sel[0]);
    if (p.renormalize) {
      sum = 0.0;
      for (int r = 0; r < p.k; ++r) sum += __shfl_sync(0xFFFFFFFFu, mine, r);
      if (lazy && nan) sum = NAN;
    }
    if (lane < p.k) {
      p.hmax[t * p.k + lane] = 0;
      p.weights[t * p.k + lane] = static_cast<float>(mine / sum * static_cast<double>(p.routed_scale));
    }
  }
}

// ---------------------------------------------------------------------------------- kernel 2

struct MoeExpertsParams {
  const uint8_t* s13;        // (E, 2 I, H / 16) scales: gate rows, then up rows
  const uint8_t* s2;         // (E, H, I / 16)
  const float* ts13;         // (E,)
  const float* ts2;
  const int* ids;
  const float* weights;
  const uint8_t* xs;         // digits of x, per token, and their row factors
  const float* x_scale;
  float* h;                  // (T k, I) hidden values (times weight and down scale)
  uint32_t* hmax;            // (T k,) bits of the largest |h| of a pair
  uint8_t* hs;               // digits of h, per pair
  float* part;               // (slices, T k, H) partial sums; part_rows rows in all
  void* y;                   // (T, H)
  uint32_t* counters;
  int T, H, I, E, k;
  int part_rows;
  int out_dtype, vec_out;
  uint32_t* err;
};

// Data written earlier in this grid: not through the read-only path.
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

struct MoePlan {
  int cnt[kMoeMaxExperts];           // pairs of an expert
  uint16_t off[kMoeMaxExperts];      // first pair of an expert in `pairs`
  uint16_t act[kMoeMaxExperts];      // experts with at least one pair, ascending
  uint16_t pairs[kMoeMaxTokens * kMoeMaxTopK];  // pairs t * k + slot, by expert
  int16_t id[kMoeMaxTokens * kMoeMaxTopK];      // expert of a pair, -1 for none
  float w[kMoeMaxTokens * kMoeMaxTopK];         // weight of a pair
  uint8_t used[kMoeMaxTokens * kMoeMaxTopK];    // the pair counts
  uint32_t totals[kMoeMaxExperts / 32];         // experts << 16 | pairs of 32 experts
  uint32_t dig[kMoeMaxExperts + 1];  // first digit task of a touched expert, and their number
  int nact;
};
constexpr int kMoeDigitBlocks = 64;  // 16-blocks of hidden values per digit task

// moe_plan for up to 32 pairs: a lane per pair of one warp (2.4 us by the whole CTA, with a barrier
// between any two steps).
__device__ __forceinline__ void moe_plan_warp(const MoeExpertsParams& p, MoePlan& pl) {
  const int lane = threadIdx.x & 31, npairs = p.T * p.k;
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  int e = -1;
  float w = 0.0f;
  if (lane < npairs) {
    e = p.ids[lane];
    w = p.weights[lane];
    if (e < 0 || e >= p.E) {
      if (e != -1) atomicOr(p.err, kErrRange);
      e = -1;
    }
  }
  // the first pair of a token that names this expert keeps the sum of the weights
  const int token = lane / p.k;
  bool first = e >= 0;
  for (int j = 0; j < npairs; ++j) {
    const int ej = __shfl_sync(kAll, e, j);
    const float wj = __shfl_sync(kAll, w, j);  // (of a later pair: still its own)
    if (j / p.k == token && ej == e) {
      if (j < lane) first = false;
      if (j > lane) w += wj;
    }
  }
  if (!first) e = -1;
  const uint32_t same = __match_any_sync(kAll, e), before = same & ((1u << lane) - 1u);
  const int cnt = __popc(same);
  const bool lead = first && before == 0;
  const uint32_t tasks =
      (static_cast<uint32_t>(cnt) * (p.I / 16) + kMoeDigitBlocks - 1) / kMoeDigitBlocks;
  int place = 0, off = 0;  // touched experts and pairs of smaller experts, and their digit tasks
  uint32_t dig = 0;
  for (int j = 0; j < npairs; ++j) {
    const int ej = __shfl_sync(kAll, e, j);
    const int cj = __shfl_sync(kAll, lead ? cnt : 0, j);
    if (cj > 0 && ej < e) {
      ++place;
      off += cj;
      dig += (static_cast<uint32_t>(cj) * (p.I / 16) + kMoeDigitBlocks - 1) / kMoeDigitBlocks;
    }
  }
  const int nact = __popc(__ballot_sync(kAll, lead));
  const uint32_t total = __reduce_add_sync(kAll, lead ? tasks : 0u);
  if (lead) {
    pl.cnt[e] = cnt;
    pl.off[e] = static_cast<uint16_t>(off);
    pl.act[place] = static_cast<uint16_t>(e);
    pl.dig[place] = dig;
  }
  if (first) {
    pl.pairs[off + __popc(before)] = static_cast<uint16_t>(lane);
    pl.w[lane] = w;
  }
  if (lane < npairs) pl.used[lane] = first;
  if (lane == 0) {
    pl.nact = nact;
    pl.dig[nact] = total;
  }
}

// Pairs by expert, by kThreads >= kMoeMaxExperts threads; pl.cnt is zero and visible before. A token
// that names an expert twice keeps the first pair with the sum of the weights; ids outside [0, E) are
// no pair (-1 quietly, others reported). Ends with a barrier.
template <int kThreads>
__device__ void moe_plan(const MoeExpertsParams& p, MoePlan& pl) {
  static_assert(kThreads >= kMoeMaxExperts, "an expert per thread");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int npairs = p.T * p.k;
  if (npairs <= 32) {
    if (warp == 0) moe_plan_warp(p, pl);
    __syncthreads();
    return;
  }
  constexpr int kPer = (kMoeMaxTokens * kMoeMaxTopK + kThreads - 1) / kThreads;
  float w[kPer] = {};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int pr = tid + i * kThreads;
    if (pr >= npairs) continue;
    int e = p.ids[pr];
    w[i] = p.weights[pr];
    if (e < 0 || e >= p.E) {
      if (e != -1) atomicOr(p.err, kErrRange);
      e = -1;
    }
    pl.id[pr] = static_cast<int16_t>(e);
    pl.w[pr] = w[i];
  }
  __syncthreads();
  int id[kPer], pos[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int pr = tid + i * kThreads;
    id[i] = -1;
    pos[i] = 0;
    if (pr >= npairs) continue;
    int e = pl.id[pr];
    const int first = pr / p.k * p.k;
    for (int s = first; s < first + p.k && e >= 0; ++s) {
      if (s == pr || pl.id[s] != e) continue;
      if (s < pr) e = -1;
      else w[i] += pl.w[s];
    }
    if (e >= 0) pos[i] = atomicAdd(&pl.cnt[e], 1);
    pl.used[pr] = e >= 0;
    id[i] = e;
  }
  __syncthreads();
  // expert of this thread: its place among the touched ones, and its first pair
  const int c = tid < p.E ? pl.cnt[tid] : 0;
  uint32_t inc = static_cast<uint32_t>(c) + (c > 0 ? 0x10000u : 0u);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31 && warp < kMoeMaxExperts / 32) pl.totals[warp] = inc;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (id[i] >= 0) pl.w[tid + i * kThreads] = w[i];
  __syncthreads();
  if (warp < kMoeMaxExperts / 32) {
    uint32_t before = 0;
    for (int i = 0; i < warp; ++i) before += pl.totals[i];
    const uint32_t end = before + inc;
    if (c > 0) {
      pl.act[(end >> 16) - 1] = static_cast<uint16_t>(tid);
      pl.off[tid] = static_cast<uint16_t>((end & 0xFFFFu) - c);
    }
    if (tid == kMoeMaxExperts - 1) pl.nact = end >> 16;
  }
  __syncthreads();
  // a pair's place in its expert's list: by its number (every CTA has the same lists)
  uint16_t* unsorted = reinterpret_cast<uint16_t*>(pl.id);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (id[i] >= 0) unsorted[pl.off[id[i]] + pos[i]] = static_cast<uint16_t>(tid + i * kThreads);
  // digit tasks before each touched expert's
  const int nact = pl.nact;
  const int mine = tid < nact ? pl.cnt[pl.act[tid]] : 0;
  const uint32_t tasks =
      (static_cast<uint32_t>(mine) * (p.I / 16) + kMoeDigitBlocks - 1) / kMoeDigitBlocks;
  uint32_t sum = tasks;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += u;
  }
  __syncthreads();  // totals is read
  if (lane == 31 && warp < kMoeMaxExperts / 32) pl.totals[warp] = sum;
  __syncthreads();
  if (warp < kMoeMaxExperts / 32) {
    uint32_t before = 0;
    for (int i = 0; i < warp; ++i) before += pl.totals[i];
    if (tid <= nact) pl.dig[tid] = before + sum - tasks;
    if (tid + 1 == nact) pl.dig[nact] = before + sum;
    if (nact == 0 && tid == 0) pl.dig[0] = 0;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (id[i] >= 0) {
      const int pr = tid + i * kThreads, o = pl.off[id[i]], n = pl.cnt[id[i]];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += unsorted[o + j] < pr ? 1 : 0;
      pl.pairs[o + rank] = static_cast<uint16_t>(pr);
    }
  __syncthreads();
}

// ---- the experts' kernel. Tasks of 256 weight rows (two MMA tiles of 128) of one expert against
// all tokens of the expert, in passes of TOK tokens; K in stages of 256:
//   gate / up: 128 hidden units, tile 0 the gate rows, tile 1 the up rows: lane i of both tiles is
//              hidden unit i. h = silu(gate) up w ts in fp32, and the pair's maximum;
//   digits:    h -> digits, once every h of an expert is there (the row factor needs the row's
//              maximum);
//   down:      256 output rows of one expert and a slice of I; partial sums per (slice, pair);
//   combine:   y = the partial sums of a token's pairs in slot order.
// Warps: 0 weight codes (TMA) and scales as they are (cp.async, 16 bytes a row); it takes the tickets
// and publishes the tasks in a queue. 1..4 the scales into the tiles tcgen05.cp wants, 64 rows each
// (4-byte cp.async straight into the tiles took 26 shared-memory cycles an instruction, 1300 of a
// stage's 2000 cycles; loads to registers three stages ahead did not cover the memory's latency).
// 5..8 activation digits, waiting for those of a down task's expert while the weights of the next
// stages already arrive. 9 MMA. 10, 11 digits of the hidden values, as experts finish. 12..19 epilogue
// and combine.
// An MMA of this kind takes about as long for 16 columns as for 128, so the weights are its 256 columns
// and the digits its 128 rows where a pass has at most 16 tokens (kSwap: half the MMAs a stage; the
// digits' sum then runs over lanes); with 24 tokens a pass the weights are two tiles of 128 rows and the
// digits 192 columns.
// Measured (the layer, GPU time, one call after another): 1 token, 8 of 64 experts of 2048 x 768: 33 us
// for 21 MB of weights: a chain of latencies (routing 5 to 9, plan 1.5, first stage 3.5, gate / up 5.5,
// epilogue and digits 6.5, down 4.5, combine 3), most of its code run once, from cold instruction caches. 7
// tokens, 6 of 128 of 4096 x 1408: 80 to 85 us (5.5 TB/s while the weights stream); 48 tokens, 8 of 128 of
// 2048 x 1024: 107 us (4.4 TB/s over this kernel); 64 tokens, 2 of 8 of 4096 x 14336: 180 to 192 us (4.6
// TB/s): there a stage's MMAs (1000 to 1250 cycles) and the drain of the one accumulator that fits tensor
// memory beside the scales take nearly as long as its bytes. A pass reads the expert's weights anew: 64
// tokens of which every one names the same two of 64 experts of 4096 x 2048 take 88 us in four passes for
// 28 MB of weights.
// Tried, no gain: a fourth stage of weights (93 us for 91 at seven tokens); scales stored to tensor
// memory from registers instead of tcgen05.cp (equal with four sets of scale words, 211 us for 199 with
// the two that fit beside 24 tokens).
constexpr int kMoeScaleWarp0 = 1, kMoeScaleWarps = 4;
constexpr int kMoeDigitWarp0 = kMoeScaleWarp0 + kMoeScaleWarps, kMoeDigitWarps = 4;
constexpr int kMoeMmaWarp = kMoeDigitWarp0 + kMoeDigitWarps;
constexpr int kMoeMakeWarp0 = kMoeMmaWarp + 1, kMoeMakeWarps = 2;
constexpr int kMoeEpiWarp0 = kMoeMakeWarp0 + kMoeMakeWarps, kMoeEpiWarps = 8;
constexpr int kMoeExpertThreads = 32 * (kMoeEpiWarp0 + kMoeEpiWarps);
constexpr int kMoeQueue = 4, kMoeStages = 3;

// 32 lanes x 16 columns of a digit sum: 20 words a lane, 16 more behind every eight lanes, so that
// neither the stores nor the loads have bank conflicts.
constexpr int kMoeSumLane = 20, kMoeSumToken = 8 * kMoeSumLane + 16;
constexpr int kMoeSumBytes = 4 * kMoeSumToken * 4;

template <int TOK>
struct MoeCfg {
  static constexpr bool kSwap = TOK <= 16;
  static constexpr int kN = kSwap ? 128 : TOK * kMoeDigitRows;  // accumulator columns of a tile
  static constexpr int kBlocks = (TOK * kMoeDigitRows + 127) / 128;  // 128-row blocks of digit scales
  static constexpr int kCodes = 2 * 128 * 128;
  static constexpr int oSw = kCodes;                         // weight scales [tile][word][512]
  static constexpr int oB = oSw + 2 * 4 * 512;               // digits
  static constexpr int oSb = oB + TOK * kMoeChunkCodes;      // digit scales [block][word][512]
  static constexpr int kStage = oSb + kBlocks * 4 * 512;
  static constexpr int kStages = kMoeStages;
  static constexpr int kRaw = 256 * 16;                      // natural weight scales of a stage
  static constexpr int oRaw = kStages * kStage;
  static constexpr int oSum = oRaw + kStages * kRaw;         // a digit sum's buffer per epilogue warp
  static constexpr int kSmem = oSum + (kSwap ? kMoeEpiWarps * kMoeSumBytes : 0) + 1024;
  static constexpr int kSfCol0 = 2 * kN;                     // after the two tiles' accumulators
  static constexpr int kSfSet = 2 * 16 + kBlocks * 16;       // scale words of a stage in tensor memory
  static_assert(kSfCol0 + 2 * kSfSet <= 512, "tensor memory budget");
  static_assert(!kSwap || TOK == 16, "128 rows of digits");
  static_assert(kStage % 1024 == 0 && oB % 1024 == 0, "1 KB swizzle atoms");
  // a full stage: the codes' tx arrive, the scale and digit warps (and the digits' bytes)
  static constexpr int kFullCount = 1 + kMoeScaleWarps + kMoeDigitWarps;
};

struct MoeCtl {
  uint64_t full[kMoeStages], empty[kMoeStages], raw_full[kMoeStages], acc_full, acc_empty;
  uint64_t qfull[kMoeQueue], qempty[kMoeQueue], drain, down_ready;
  uint32_t queue[kMoeQueue];
  uint32_t abort_flag, tmem_base;
  uint32_t warps;  // epilogue warps that finished their part of a down task
  uint32_t digits_seen;  // down tasks whose digits are there, or kMoeAllSeen
};
constexpr int kMoeQueueReaders = kMoeScaleWarps + kMoeDigitWarps + 1 + kMoeEpiWarps;

// A queue entry: phase in the top two bits (0 gate / up, 1 down, 2 end), task below.
struct MoeTask {
  uint32_t phase, index;
};

// Geometry of a task.
struct MoeGeom {
  int a, e, cnt, off;   // touched expert, expert, its pairs
  int c0, c1;           // stages of K
  int K, row0, z;       // first hidden unit / output row, slice
  int64_t ra, rb;       // first weight rows of the two tiles
  bool two;             // the second tile exists
};
struct MoeShape {
  int blocks1, blocks2, slices;
  uint32_t total1, total2;
  __device__ __forceinline__ MoeGeom geom(const MoeExpertsParams& p, const MoePlan& pl,
                                          const MoeTask& t) const {
    MoeGeom g;
    if (t.phase == 0) {
      g.a = t.index / blocks1;
      g.e = pl.act[g.a];
      g.row0 = (t.index % blocks1) * 128;
      g.z = 0;
      g.c0 = 0;
      g.c1 = (p.H + 255) / 256;
      g.K = p.H;
      g.ra = static_cast<int64_t>(g.e) * 2 * p.I + g.row0;
      g.rb = g.ra + p.I;
      g.two = true;
    } else {
      const int ab = t.index / slices;
      g.z = t.index % slices;
      g.a = ab / blocks2;
      g.e = pl.act[g.a];
      g.row0 = (ab % blocks2) * 256;
      const int n = (p.I + 255) / 256;
      g.c0 = n * g.z / slices;
      g.c1 = n * (g.z + 1) / slices;
      g.K = p.I;
      g.ra = static_cast<int64_t>(g.e) * p.H + g.row0;
      g.rb = g.ra + 128;
      g.two = g.row0 + 128 < p.H;
    }
    g.cnt = pl.cnt[g.e];
    g.off = pl.off[g.e];
    return g;
  }
};

// A whole warp's bounded wait: the same answer in every lane.
__device__ __forceinline__ bool moe_warp_wait(uint64_t& bar, uint32_t parity, uint32_t code,
                                              MoeCtl& ctl, uint32_t* err) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&bar), parity, err, code, &ctl.abort_flag));
}

// The next queue entry (the shuffle waits for the read before the release).
__device__ __forceinline__ bool moe_next_task(MoeTask& t, RingPos<kMoeQueue>& q, MoeCtl& ctl,
                                              uint32_t* err) {
  if (!moe_warp_wait(ctl.qfull[q.slot], q.phase, kErrWaitTma, ctl, err)) return false;
  uint32_t v = *reinterpret_cast<volatile uint32_t*>(&ctl.queue[q.slot]);
  v = __shfl_sync(0xFFFFFFFFu, v, 0);
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl.qempty[q.slot]));
  q.next();
  t.phase = v >> 30;
  t.index = v & 0x3FFFFFFFu;
  return true;
}

// A whole warp: until *counter >= target (counter of this grid, or kCta of this CTA), bounded; `seen` is
// the value that ended the lane's wait, and only that one was acquired. A counter
// of the grid is read again only after a pause: a poll takes its turn in the same L2 slice as the
// additions it waits for. (One warp per CTA polls for the others where they wait for the same: with all
// eight epilogue warps of 148 CTAs polling, the combine phase began 1.5 us later.)
template <bool kCta>
__device__ __forceinline__ bool moe_wait(const uint32_t* counter, uint32_t target, MoeCtl& ctl,
                                         uint32_t* err, uint32_t& seen) {
  bool ok = true;
  const long long c0 = clock64();
  while (true) {
    if constexpr (kCta)
      asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];"
                   : "=r"(seen)
                   : "r"(smem_u32(counter))
                   : "memory");
    else
      seen = ld_acquire_gpu(counter);
    if (seen >= target) break;
    if (*reinterpret_cast<volatile uint32_t*>(&ctl.abort_flag)) {
      ok = false;
      break;
    }
    if (static_cast<unsigned long long>(clock64() - c0) > kWaitLimitCycles) {
      atomicOr(err, kErrWaitOperand);
      *reinterpret_cast<volatile uint32_t*>(&ctl.abort_flag) = 1u;
      ok = false;
      break;
    }
    __nanosleep(kCta ? 20 : 60);
  }
  return __all_sync(0xFFFFFFFFu, ok);
}
template <bool kCta>
__device__ __forceinline__ bool moe_wait(const uint32_t* counter, uint32_t target, MoeCtl& ctl,
                                         uint32_t* err) {
  uint32_t seen;
  return moe_wait<kCta>(counter, target, ctl, err, seen);
}
constexpr uint32_t kMoeAllSeen = 1u << 30;

// A warp's stores, then the count (lane 0's release covers what the others stored before the
// __syncwarp).
__device__ __forceinline__ void moe_count(uint32_t* counter) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
}

__device__ __forceinline__ uint32_t moe_ticket(uint32_t* counter) {
  uint32_t k = 0;
  if ((threadIdx.x & 31) == 0) k = atomicAdd(counter, 1u);
  return __shfl_sync(0xFFFFFFFFu, k, 0);
}
// An epilogue warp's part of a down task is done: its stores before the count. The last of eight
// parts counts for the CTA (parts of two tasks may mix; the phase's total is what is waited for).
__device__ __forceinline__ void moe_count_down(uint32_t* counter, uint32_t* warps) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    uint32_t before;
    asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;"
                 : "=r"(before)
                 : "r"(smem_u32(warps))
                 : "memory");
    if ((before & (kMoeEpiWarps - 1)) == kMoeEpiWarps - 1)
      asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
  }
}

// Sum of a token's digit columns, digit p times 8^-p (the product by 1/8 is exact).
__device__ __forceinline__ float moe_sum8(const uint32_t* r) {
  float s = __uint_as_float(r[kMoeDigitCount - 1]);
#pragma unroll
  for (int p = kMoeDigitCount - 2; p >= 0; --p) s = fmaf(s, 0.125f, __uint_as_float(r[p]));
  return s;
}

// 16 columns of eight lanes' digits: lane c of the eight gets the sums over them (digit p times 8^-p) of
// columns 2 c and 2 c + 1, by way of shared memory. (In registers, by three exchanges of halves, it took 14 shuffles
// and 28 selects: with one to four tokens all of that is the work of one scheduler's warps, and the
// accumulator is busy until it ends.)
__device__ __forceinline__ float2 moe_lane_sums(const uint32_t (&d)[16], float* buf) {
  const int lane = threadIdx.x & 31;
  float* own = buf + (lane >> 3) * kMoeSumToken;
  uint4* dst = reinterpret_cast<uint4*>(own + (lane & 7) * kMoeSumLane);
  if ((lane & 7) < kMoeDigitCount) {
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = make_uint4(d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]);
  }
  __syncwarp();
  const float2* src = reinterpret_cast<const float2*>(own) + (lane & 7);
  float2 v[kMoeDigitCount];
#pragma unroll
  for (int p = 0; p < kMoeDigitCount; ++p) v[p] = src[p * (kMoeSumLane / 2)];
  __syncwarp();
#pragma unroll
  for (int p = kMoeDigitCount - 2; p >= 0; --p) {
    v[p].x = fmaf(v[p + 1].x, 0.125f, v[p].x);
    v[p].y = fmaf(v[p + 1].y, 0.125f, v[p].y);
  }
  return v[0];
}

// Four scale words (a row's 16 scales of a stage) into their tiles, 512 bytes apart.
__device__ __forceinline__ void moe_store_scales(uint32_t dst, const uint2& lo, const uint2& hi) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(lo.x) : "memory");
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + 512), "r"(lo.y) : "memory");
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + 1024), "r"(hi.x) : "memory");
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + 1536), "r"(hi.y) : "memory");
}
// A scale warp's part of a stage is stored: the tensor core reads it through the async proxy.
__device__ __forceinline__ void moe_scales_ready(uint64_t& full) {
  fence_proxy_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&full));
}
constexpr int kMoeAhead = 3;  // stages whose scales are in registers

template <int TOK>
__global__ void __launch_bounds__(kMoeExpertThreads, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap tm_w13,
                       const __grid_constant__ CUtensorMap tm_w2, const MoeExpertsParams p) {
  using Cfg = MoeCfg<TOK>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ MoePlan pl;
  __shared__ MoeCtl ctl;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  if (tid == 0) {
    ctl.abort_flag = 0;
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(smem_u32(&ctl.full[s]), Cfg::kFullCount);
      mbar_init(smem_u32(&ctl.empty[s]), 1);
      mbar_init(smem_u32(&ctl.raw_full[s]), 32);
    }
    mbar_init(smem_u32(&ctl.acc_full), 1);
    mbar_init(smem_u32(&ctl.acc_empty), kMoeEpiWarps);
    for (int s = 0; s < kMoeQueue; ++s) {
      mbar_init(smem_u32(&ctl.qfull[s]), 1);
      mbar_init(smem_u32(&ctl.qempty[s]), kMoeQueueReaders);
    }
    mbar_init(smem_u32(&ctl.drain), 1);
    mbar_init(smem_u32(&ctl.down_ready), 1);
    ctl.warps = 0;
    ctl.digits_seen = 0;
    fence_mbar_init();
  }
  if (warp == kMoeMmaWarp) {
    tmem_alloc(smem_u32(&ctl.tmem_base), 512);
    tmem_relinquish();
  }
  for (int e = tid; e < p.E; e += kMoeExpertThreads) pl.cnt[e] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = ctl.tmem_base;
  grid_dep_wait();
  uint32_t first_ticket = 0;  // taken while the plan is made
  if (tid == 0) first_ticket = atomicAdd(p.counters + kMoeGateUp, 1u);
  moe_plan<kMoeExpertThreads>(p, pl);
  const int nact = pl.nact;

  MoeShape sh;
  sh.blocks1 = p.I / 128;
  sh.total1 = static_cast<uint32_t>(nact) * sh.blocks1;
  sh.blocks2 = (p.H + 255) / 256;
  // slices of I per down task: while the tasks do not fill the grid and the partials fit
  sh.slices = 1;
  while (nact * sh.blocks2 * sh.slices < static_cast<int>(gridDim.x) &&
         2 * sh.slices * p.T * p.k <= p.part_rows && p.I / 256 >= 2 * sh.slices)
    sh.slices *= 2;
  sh.total2 = static_cast<uint32_t>(nact) * sh.blocks2 * sh.slices;
  const int blocks_h = p.I / 16;
  const uint32_t total_d = pl.dig[nact];
  uint32_t* gate_up_done = p.counters + kMoeCounters;
  uint32_t* digits_done = gate_up_done + p.E;

  RingPos<kMoeQueue> q;
  RingPos<Cfg::kStages> r;
  MoeTask t;
  if (warp == 0) {
    // -------------------------------------------------------------------- weight codes, tickets
    if (lane == 0) {
      prefetch_tmap(&tm_w13);
      prefetch_tmap(&tm_w2);
    }
    uint32_t phase = 0;
    bool ok = true, first = true;
    while (ok) {
      // the next task: the phase's tickets, then the next phase's
      t.phase = 2;
      t.index = 0;
      while (phase < 2) {
        uint32_t k;
        if (first) {
          k = __shfl_sync(0xFFFFFFFFu, first_ticket, 0);
          first = false;
        } else {
          k = moe_ticket(p.counters + (phase == 0 ? kMoeGateUp : kMoeDown));
        }
        if (k < (phase == 0 ? sh.total1 : sh.total2)) {
          t.phase = phase;
          t.index = k;
          break;
        }
        ++phase;
      }
      if (!(ok = moe_warp_wait(ctl.qempty[q.slot], q.phase ^ 1u, kErrWaitEmpty, ctl, p.err))) break;
      if (lane == 0) {
        ctl.queue[q.slot] = t.phase << 30 | t.index;
        mbar_arrive(smem_u32(&ctl.qfull[q.slot]));
      }
      q.next();
      if (t.phase == 2) break;
      const MoeGeom gm = sh.geom(p, pl, t);
      const CUtensorMap* tm = t.phase == 0 ? &tm_w13 : &tm_w2;
      const int pitch = gm.K / 16, half = 8 * (lane & 1);
      const uint8_t* base = (t.phase == 0 ? p.s13 : p.s2) + (lane >> 1) * pitch + half;
      const uint8_t *sa = base + gm.ra * pitch, *sb = base + gm.rb * pitch;
      if (lane < (gm.two ? 2 : 1)) {  // all of the task's scales towards L2: 16 bytes a row come slowly
        const uint8_t* rows = (t.phase == 0 ? p.s13 : p.s2) + (lane == 0 ? gm.ra : gm.rb) * pitch;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                         reinterpret_cast<uint64_t>(rows) & ~15ull),
                     "r"(128 * pitch)
                     : "memory");
      }
      for (int n0 = 0; n0 < gm.cnt && ok; n0 += TOK)
        for (int c = gm.c0; c < gm.c1; ++c) {
          // (an empty stage's raw scales are read too: they were repacked before its MMAs)
          if (!(ok = moe_warp_wait(ctl.empty[r.slot], r.phase ^ 1u, kErrWaitEmpty, ctl, p.err))) break;
          if (lane == 0) {
            const uint32_t st = smem_u32(smem + r.slot * Cfg::kStage);
            const uint32_t fb = smem_u32(&ctl.full[r.slot]);
            mbar_arrive_expect_tx(fb, gm.two ? Cfg::kCodes : Cfg::kCodes / 2);
            tma_load_2d(st, tm, c * 128, static_cast<int32_t>(gm.ra), fb);
            if (gm.two)
              tma_load_2d(st + Cfg::kCodes / 2, tm, c * 128, static_cast<int32_t>(gm.rb), fb);
          }
          __syncwarp();
          if (c * 16 + half < pitch) {  // the last stage may have 8 scales a row
            const uint32_t dst = smem_u32(smem + Cfg::oRaw + r.slot * Cfg::kRaw) + 8 * lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + 256 * i),
                           "l"(sa + c * 16 + 16 * i * pitch)
                           : "memory");
              if (gm.two)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + 2048 + 256 * i),
                             "l"(sb + c * 16 + 16 * i * pitch)
                             : "memory");
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                           smem_u32(&ctl.raw_full[r.slot]))
                       : "memory");
          r.next();
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp < kMoeDigitWarp0) {
    // ---------------------------------------- weight scales into their tiles: half the rows of a tile
    // Lane (i, j) = (lane / 8, lane % 8) takes rows 32 i + 16 h + j and + 8, h the half: the four row
    // groups of one j are side by side in a tile, so neither loads nor stores have bank conflicts.
    const int m = (warp - kMoeScaleWarp0) >> 1;
    const int row = 32 * (lane >> 3) + 16 * ((warp - kMoeScaleWarp0) & 1) + (lane & 7);
    const uint32_t at = Cfg::oSw + m * 2048 + (row & 31) * 16 + (row >> 5) * 4;
    while (moe_next_task(t, q, ctl, p.err) && t.phase != 2) {
      const MoeGeom gm = sh.geom(p, pl, t);
      bool ok = true;
      for (int n0 = 0; n0 < gm.cnt && ok; n0 += TOK)
        for (int c = gm.c0; c < gm.c1; ++c) {
          if (!(ok = moe_warp_wait(ctl.raw_full[r.slot], r.phase, kErrWaitTma, ctl, p.err))) break;
          const uint8_t* raw = smem + Cfg::oRaw + r.slot * Cfg::kRaw + m * 2048 + row * 16;
          const uint4 lo = *reinterpret_cast<const uint4*>(raw);
          const uint4 hi = *reinterpret_cast<const uint4*>(raw + 128);
          // (raw scales arrive only in a stage whose MMAs are done: its tiles are free)
          const uint32_t dst = smem_u32(smem + r.slot * Cfg::kStage) + at;
          moe_store_scales(dst, make_uint2(lo.x, lo.y), make_uint2(lo.z, lo.w));
          moe_store_scales(dst + 128, make_uint2(hi.x, hi.y), make_uint2(hi.z, hi.w));
          moe_scales_ready(ctl.full[r.slot]);
          r.next();
        }
      if (!ok) break;
    }
  } else if (warp < kMoeMmaWarp) {
    // ---------------------------------------------------------------- activation digits and scales
    // Warp `part`: tokens part + 4 i. Scales: lane = 8 i + digit, again the four row groups of a line
    // side by side.
    const int part = warp - kMoeDigitWarp0;
    constexpr int kSets = Cfg::kBlocks;
    bool ready = false;  // the digits of all experts
    uint32_t seen = 0;
    while (moe_next_task(t, q, ctl, p.err) && t.phase != 2) {
      const MoeGeom gm = sh.geom(p, pl, t);
      if (t.phase == 1 && !ready) {
        ++seen;
        if (part == 0) {
          ready = __all_sync(0xFFFFFFFFu, ld_acquire_gpu(p.counters + kMoeDigitsDone) >= total_d);
          if (!ready &&
              !moe_wait<false>(digits_done + gm.a, pl.dig[gm.a + 1] - pl.dig[gm.a], ctl, p.err))
            break;
          if (lane == 0)
            asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(&ctl.digits_seen)),
                         "r"(ready ? kMoeAllSeen : seen)
                         : "memory");
        } else {
          uint32_t now;
          if (!moe_wait<true>(&ctl.digits_seen, seen, ctl, p.err, now)) break;
          ready = __all_sync(0xFFFFFFFFu, now == kMoeAllSeen);
        }
        // written by ordinary stores of this grid; the bulk copies read through the async proxy
        asm volatile("fence.proxy.async;" ::: "memory");
      }
      const uint8_t* base = t.phase == 0 ? p.xs : p.hs;
      bool ok = true;
      for (int n0 = 0; n0 < gm.cnt && ok; n0 += TOK) {
        const int n = min(gm.cnt - n0, TOK);
        auto image = [&](int i) {
          const int pr = pl.pairs[gm.off + n0 + i];
          return base + (t.phase == 0 ? pr / p.k : pr) * moe_image_row(gm.K);
        };
        // codes of tokens part + 4 lane
        const uint8_t* codes = part + 4 * lane < n ? image(part + 4 * lane) : nullptr;
        const uint32_t code_bytes = (n - part + 3) / 4 * kMoeChunkCodes;
        const uint8_t* src[kSets];
        uint32_t at[kSets];
        uint4 w[kMoeAhead][kSets];
#pragma unroll
        for (int k = 0; k < kSets; ++k) {
          const int i = 16 * k + part + 4 * (lane >> 3);
          src[k] = i < n && i < TOK ? image(i) + kMoeChunkCodes + 16 * (lane & 7) : nullptr;
          at[k] = Cfg::oSb + k * 2048 + (part * 8 + (lane & 7)) * 16 + (lane >> 3) * 4;
        }
        auto load = [&](uint4 (&v)[kSets], int c) {
#pragma unroll
          for (int k = 0; k < kSets; ++k)
            if (src[k] != nullptr && c < gm.c1) v[k] = ld_cg(src[k] + static_cast<int64_t>(c) * kMoeChunk);
        };
#pragma unroll
        for (int j = 0; j < kMoeAhead; ++j) load(w[j], gm.c0 + j);
        for (int c0 = gm.c0; c0 < gm.c1 && ok; c0 += kMoeAhead) {
#pragma unroll
          for (int j = 0; j < kMoeAhead; ++j) {
            if (c0 + j >= gm.c1) break;
            if (!(ok = moe_warp_wait(ctl.empty[r.slot], r.phase ^ 1u, kErrWaitEmpty, ctl, p.err))) break;
            const uint32_t st = smem_u32(smem + r.slot * Cfg::kStage);
            const uint32_t fb = smem_u32(&ctl.full[r.slot]);
            if (lane == 0)
              asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(fb),
                           "r"(code_bytes)
                           : "memory");
            __syncwarp();
            if (codes != nullptr)
              bulk_load(st + Cfg::oB + (part + 4 * lane) * kMoeChunkCodes,
                        codes + static_cast<int64_t>(c0 + j) * kMoeChunk, kMoeChunkCodes, fb);
#pragma unroll
            for (int k = 0; k < kSets; ++k)
              if (src[k] != nullptr)
                moe_store_scales(st + at[k], make_uint2(w[j][k].x, w[j][k].y),
                                 make_uint2(w[j][k].z, w[j][k].w));
            moe_scales_ready(ctl.full[r.slot]);
            load(w[j], c0 + j + kMoeAhead);
            r.next();
          }
        }
      }
      if (!ok) break;
    }
  } else if (warp == kMoeMmaWarp) {
    // ----------------------------------------------------------------------------------- MMA
    uint32_t aph = 0, set = 0;
    bool ok = true;
    while (ok && moe_next_task(t, q, ctl, p.err) && t.phase != 2) {
      const MoeGeom gm = sh.geom(p, pl, t);
      for (int n0 = 0; n0 < gm.cnt && ok; n0 += TOK) {
        const int n = min(gm.cnt - n0, TOK);
        const uint32_t N = Cfg::kSwap ? (gm.two ? 256u : 128u)
                                      : static_cast<uint32_t>(n * kMoeDigitRows + 15) & ~15u;
        const uint32_t idesc = idesc_mxf4(128, N, false, 0);
        const int blocks = !Cfg::kSwap && N > 128 ? 2 : 1;
        if (!(ok = moe_warp_wait(ctl.acc_empty, aph ^ 1u, kErrWaitAccum, ctl, p.err))) break;
        aph ^= 1u;
        tc_fence_after();
        for (int c = gm.c0; c < gm.c1; ++c) {
          if (!(ok = moe_warp_wait(ctl.full[r.slot], r.phase, kErrWaitTma, ctl, p.err))) break;
          tc_fence_after();
          const uint32_t st = smem_u32(smem + r.slot * Cfg::kStage);
          // scale words in tensor memory: weights [word][tile] (kSwap: one 256-row operand) or
          // [tile][word], digits [word][block]
          const uint32_t sfw = tb + Cfg::kSfCol0 + set * Cfg::kSfSet, sfd = sfw + 32;
          constexpr uint32_t kWord = Cfg::kSwap ? 8 : 4, kTile = Cfg::kSwap ? 4 : 16;
          const int steps = min(4, gm.K / 64 - c * 4);
          if (elect_one()) {
            for (int kk = 0; kk < steps; ++kk) {
              tmem_cp_32x128b_x4(sfw + kWord * kk, sdesc_sf(st + Cfg::oSw + kk * 512));
              if (gm.two)
                tmem_cp_32x128b_x4(sfw + kWord * kk + kTile, sdesc_sf(st + Cfg::oSw + (4 + kk) * 512));
              tmem_cp_32x128b_x4(sfd + kk * 4 * Cfg::kBlocks, sdesc_sf(st + Cfg::oSb + kk * 512));
              if (Cfg::kBlocks > 1 && blocks > 1)
                tmem_cp_32x128b_x4(sfd + kk * 4 * Cfg::kBlocks + 4,
                                   sdesc_sf(st + Cfg::oSb + 2048 + kk * 512));
            }
            for (int kk = 0; kk < steps; ++kk) {
              const uint32_t accumulate = (c > gm.c0 || kk > 0) ? 1u : 0u;
              const uint64_t wd = sdesc_sw128(st + kk * 32), dd = sdesc_sw128(st + Cfg::oB + kk * 32);
              const uint32_t sd = sfd + kk * 4 * Cfg::kBlocks;
              if constexpr (Cfg::kSwap) {
                mma_mxf4_ss<true, false>(tb, dd, wd, idesc, sd, sfw + kWord * kk, accumulate);
              } else {
                mma_mxf4_ss<true, false>(tb, wd, dd, idesc, sfw + kWord * kk, sd, accumulate);
                if (gm.two)
                  mma_mxf4_ss<true, false>(tb + Cfg::kN, sdesc_sw128(st + Cfg::kCodes / 2 + kk * 32),
                                           dd, idesc, sfw + kWord * kk + kTile, sd, accumulate);
              }
            }
            tc_commit(smem_u32(&ctl.empty[r.slot]));
            if (c + 1 == gm.c1) tc_commit(smem_u32(&ctl.acc_full));
          }
          __syncwarp();
          r.next();
          set ^= 1u;
        }
      }
    }
    // arrives once every tcgen05 operation this warp issued has completed
    if (elect_one()) tc_commit(smem_u32(&ctl.drain));
    __syncwarp();
    mbar_wait(smem_u32(&ctl.drain), 0, p.err, kErrWaitMma, nullptr);
  } else if (warp < kMoeEpiWarp0) {
    // ------------------------------------------------------------- digits of the hidden values
    while (true) {
      const uint32_t k = moe_ticket(p.counters + kMoeDigits);
      if (k >= total_d) break;
      int a = 0;
      for (int hi = nact; hi - a > 1;) {  // dig[a] <= k < dig[a + 1]
        const int mid = (a + hi) >> 1;
        if (pl.dig[mid] <= k) a = mid;
        else hi = mid;
      }
      if (!moe_wait<false>(gate_up_done + a, sh.blocks1 * kMoeEpiWarps, ctl, p.err)) break;
      const int e = pl.act[a];
#pragma unroll 1
      for (int i = 0; i < kMoeDigitBlocks; i += 32) {
        const int b = static_cast<int>(k - pl.dig[a]) * kMoeDigitBlocks + i + lane;
        if (b < pl.cnt[e] * blocks_h) {  // a multiple of eight
          const int pr = pl.pairs[pl.off[e] + b / blocks_h], blk = b % blocks_h;
          const float up = pow2f(moe_row_shift(__ldcg(p.hmax + pr)));
          const float* src = p.h + static_cast<int64_t>(pr) * p.I + 16 * blk;
          float v[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 u = ld_cg(src + 4 * j);
            v[4 * j] = __uint_as_float(u.x) * up;
            v[4 * j + 1] = __uint_as_float(u.y) * up;
            v[4 * j + 2] = __uint_as_float(u.z) * up;
            v[4 * j + 3] = __uint_as_float(u.w) * up;
          }
          moe_digits(v, p.hs + pr * moe_image_row(p.I), blk);
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");
      moe_count(digits_done + a);
      moe_count(p.counters + kMoeDigitsDone);
    }
  } else {
    // ------------------------------------------------------------------------------ epilogue
    const int group = (warp - kMoeEpiWarp0) / 4, quarter = warp & 3;
    const int row = 32 * quarter + lane;  // row of the MMA tile
    const uint32_t acc = tb + (static_cast<uint32_t>(32 * quarter) << 16);
    uint32_t aph = 0;
    bool ok = true;
    while ((ok = moe_next_task(t, q, ctl, p.err)) && t.phase != 2) {
      const MoeGeom gm = sh.geom(p, pl, t);
      const float ts13 = p.ts13[gm.e], ts2 = p.ts2[gm.e];
      for (int n0 = 0; n0 < gm.cnt; n0 += TOK) {
        const int n = min(gm.cnt - n0, TOK);
        // what the tokens need besides, by lane: loaded before the wait
        const bool up = t.phase == 0;
        float f0 = 0.0f, f1 = 0.0f;
        int pr_l = 0;
        if (lane < n) {
          pr_l = pl.pairs[gm.off + n0 + lane];
          if (up) {
            f0 = p.x_scale[pr_l / p.k] * ts13;
            f1 = pl.w[pr_l] * ts2;
          }
        }
        if (!(ok = moe_warp_wait(ctl.acc_full, aph, kErrWaitAccum, ctl, p.err))) break;
        aph ^= 1u;
        // (a pair's maximum is final once its expert's down product runs, not before)
        if (!up && lane < n) f0 = moe_row_factor(__ldcg(p.hmax + pr_l));
        tc_fence_after();
        auto release = [&]() {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctl.acc_empty));
        };
        if constexpr (Cfg::kSwap) {
          // Lanes 8 i .. 8 i + 7 of a quarter: the digits of token 4 quarter + i; columns: weight
          // rows. Up: this group of four warps takes 64 hidden units, both tiles; down: the 128
          // rows of its own tile. Four pieces of 16 + 16 columns, summed over the digits so that
          // lane p of eight ends with columns 2 p and 2 p + 1 of each 16.
          const int c = 4 * quarter + (lane >> 3);
          const bool work = 4 * quarter < n && (up || group == 0 || gm.two);
          // piece i of eight: 16 columns of the first tile (even i) or the second; a piece is loaded while
          // the one before is summed
          float2 v[8];
          if (work) {
            float* buf = reinterpret_cast<float*>(smem + Cfg::oSum) +
                         (warp - kMoeEpiWarp0) * (kMoeSumBytes / 4);
            uint32_t d[2][16];
            auto load = [&](int i) {
              tmem_ld_x16(acc + (up ? 128 * (i & 1) + 64 * group + 16 * (i >> 1) : 128 * group + 16 * i),
                          d[i & 1]);
            };
            load(0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              tmem_ld_wait_x16(d[i & 1]);
              if (i < 7) load(i + 1);
              v[i] = moe_lane_sums(d[i & 1], buf);
            }
          }
          release();
          if (work) {
            const int pr = __shfl_sync(0xFFFFFFFFu, pr_l, c);
            const float g0 = __shfl_sync(0xFFFFFFFFu, f0, c), g1 = __shfl_sync(0xFFFFFFFFu, f1, c);
            uint32_t hm = 0;
            float* dst = up ? p.h + static_cast<int64_t>(pr) * p.I + gm.row0 + 64 * group
                            : p.part + (static_cast<int64_t>(gm.z) * p.T * p.k + pr) * p.H + gm.row0 +
                                  128 * group;
            float2* out = reinterpret_cast<float2*>(dst) + (lane & 7);
            if (c < n) {
              if (up) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float2 g = v[2 * j], u = v[2 * j + 1];
                  const float2 h = make_float2(silu_rn(g.x * g0) * (u.x * g0) * g1,
                                               silu_rn(g.y * g0) * (u.y * g0) * g1);
                  out[8 * j] = h;
                  hm = max(hm, max(__float_as_uint(h.x) & 0x7FFFFFFFu, __float_as_uint(h.y) & 0x7FFFFFFFu));
                }
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) out[8 * i] = make_float2(v[i].x * g0, v[i].y * g0);
              }
            }
            if (up) {
#pragma unroll
              for (int o = 1; o < 8; o <<= 1) hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, o));
              if ((lane & 7) == 0 && c < n) atomicMax(p.hmax + pr, hm);
            }
          }
        } else {
          // Lane: weight row; columns: the tokens' digits. Up: this group of four warps takes every
          // other token, both tiles; down: all tokens of its own tile.
          float sum[TOK];
#pragma unroll
          for (int j = 0; j < TOK / 2; ++j) {
            const int c = up ? 2 * j + group : 2 * j;
            if (c < n && (up || group == 0 || gm.two)) {
              uint32_t d0[8], d1[8];
              tmem_ld_x8(acc + (up ? 0 : group * Cfg::kN) + c * kMoeDigitRows, d0);
              tmem_ld_x8(acc + (up ? Cfg::kN + c * kMoeDigitRows
                                   : group * Cfg::kN + (c + 1) * kMoeDigitRows), d1);
              tmem_ld_wait_x8(d0);
              tmem_ld_wait_x8(d1);
              sum[2 * j] = moe_sum8(d0);
              sum[2 * j + 1] = moe_sum8(d1);
            }
          }
          release();
          if (up) {
#pragma unroll
            for (int j = 0; j < TOK / 2; ++j) {
              const int c = 2 * j + group;
              if (c >= n) break;
              const int pr = __shfl_sync(0xFFFFFFFFu, pr_l, c);
              const float s = __shfl_sync(0xFFFFFFFFu, f0, c), wt = __shfl_sync(0xFFFFFFFFu, f1, c);
              const float h = silu_rn(sum[2 * j] * s) * (sum[2 * j + 1] * s) * wt;
              p.h[static_cast<int64_t>(pr) * p.I + gm.row0 + row] = h;
              const uint32_t hm =
                  __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(h) & 0x7FFFFFFFu);
              if (lane == 0) atomicMax(p.hmax + pr, hm);
            }
          } else if (group == 0 || gm.two) {
            float* dst = p.part + static_cast<int64_t>(gm.z) * p.T * p.k * p.H + gm.row0 + 128 * group + row;
#pragma unroll
            for (int c = 0; c < TOK; ++c) {
              if (c >= n) break;
              dst[static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, pr_l, c)) * p.H] =
                  sum[c] * __shfl_sync(0xFFFFFFFFu, f0, c);
            }
          }
        }
      }
      if (!ok) break;
      if (t.phase == 0) moe_count(gate_up_done + gm.a);
      else moe_count_down(p.counters + kMoeDownDone, &ctl.warps);
    }

    // combine: 128 outputs of a token per warp and turn, dealt by index (no one waits for these),
    // eight partial sums in flight
    const int blocks3 = p.H / 128, terms = p.k * sh.slices;
    const int slice_bits = 31 - __clz(sh.slices);  // a power of two
    if (warp == kMoeEpiWarp0) {
      ok = ok && moe_wait<false>(p.counters + kMoeDownDone, sh.total2, ctl, p.err);
      if (ok && lane == 0) mbar_arrive(smem_u32(&ctl.down_ready));
    } else {
      ok = ok && moe_warp_wait(ctl.down_ready, 0, kErrWaitOperand, ctl, p.err);
    }
    for (int task = blockIdx.x + gridDim.x * (warp - kMoeEpiWarp0); ok && task < p.T * blocks3;
         task += gridDim.x * kMoeEpiWarps) {
      const int tok = task / blocks3, h0 = (task % blocks3) * 128 + 4 * lane;
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int i0 = 0; i0 < terms; i0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = i0 + j, s = i >> slice_bits, z = i & (sh.slices - 1);
          const int pr = tok * p.k + s;
          v[j] = i < terms && pl.used[pr]
                     ? ld_cg(p.part + (static_cast<int64_t>(z) * p.T * p.k + pr) * p.H + h0)
                     : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[0] += __uint_as_float(v[j].x);
          o[1] += __uint_as_float(v[j].y);
          o[2] += __uint_as_float(v[j].z);
          o[3] += __uint_as_float(v[j].w);
        }
      }
      store_row<4>(p.y, static_cast<int64_t>(tok) * p.H + h0, o, p.out_dtype, p.vec_out);
    }
  }
  // ------------------------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  // A wait ran out: what this warp issued last to each slot (weights; digits) lands before the CTA exits.
  // Limited: a slot that another role never arrived at does not complete, but its copies do land.
  if (*abort_flag && (warp == 0 || (warp >= kMoeDigitWarp0 && warp < kMoeMmaWarp))) {
    for (int s = 0; s < Cfg::kStages; ++s)
      mbar_wait(smem_u32(&ctl.full[s]), r.last_parity(s), p.err, kErrWaitTma, nullptr,
                kWaitLimitCycles / 8);
  }
  __syncthreads();
  if (warp == kMoeMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tb, 512);
  }
}

}  // namespace bd
