// moe.cuh -- a mixture-of-experts layer for a few tokens (T <= 64) in two kernels, expert weights
// in NVFP4 as bd_quantize_b_nvfp4 writes them (natural codes and scales, nothing packed):
//
//   logits = x Wr^T;  s = softmax or sigmoid(logits);  top-k by s (+ bias);  w = s (renormalised)
//   y_t = sum over the chosen experts e of w_e * Wd_e (silu(Wg_e x_t) * (Wu_e x_t))
//
// A few tokens read far more weights than they compute with, so the experts' kernel streams the
// touched experts' 4-bit weights once through a ring in shared memory (TMA), turns them into fp16
// MMA fragments in registers (exactly: an E2M1 times an E4M3 value has at most 6 significant bits)
// and multiplies by all tokens of the expert with mma.sync (weights are the 16 rows, tokens the 8
// columns; the tensor work is far below what the weights' bytes cost, so the legacy MMA, whose
// fragments come from registers, saves the trip of converted weights through shared memory).
// Activations are fp16 images with a power-of-two scale per token and 128 elements: exact for x
// (down to 2^-29 of a token's largest value), one rounding to 11 bits for the hidden values. Sums
// are fp32.
//
// Kernel 1 (moe_route_kernel, or moe_prepare_kernel where the caller brings the routing): router
// products, selection, image of x, counters to zero.
// Kernel 2 (moe_experts_kernel): gate / up, down and combine phases in one grid. Work is handed out
// by tickets (atomic counters), all tasks of a phase before those of the next: a CTA that waits for a
// phase to finish knows that each of its tasks is held by a CTA that already runs, so the wait ends
// without any guarantee that the whole grid is resident at once.
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

// Image of a row of activations: per 128 elements 256 bytes of fp16, one fp32 factor (what the fp16
// values are multiplied by) and 12 unused bytes. A thread of an MMA lane quad q takes elements
// 32 q .. 32 q + 31 of a block (one 16-byte piece of the weights' codes) in four loads of 8; (q, load)
// are exchanged so that a quad's load is 64 contiguous bytes.
constexpr int kMoeBlock = 272;
__host__ __device__ __forceinline__ int moe_image_offset(int k) {  // bytes, of element k
  const int r = k & 127;
  return (k >> 7) * kMoeBlock + ((r >> 3) & 3) * 64 + (r >> 5) * 16 + (r & 7) * 2;
}
__host__ __device__ __forceinline__ int64_t moe_image_row(int K) {
  return static_cast<int64_t>(K / 128) * kMoeBlock;
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
  uint8_t* xs;             // images of x
  uint32_t* counters;
  int T, H, E, k;
  int sigmoid, renormalize;
  float routed_scale;
};

// Exponent that takes values whose largest magnitude has these bits to [2^14, 2^15): times
// 2^(14 - E). A NaN or Inf stays one under E = 14.
__device__ __forceinline__ int moe_exp(uint32_t amax_bits) {
  return amax_bits >= 0x7F800000u ? 14 : max(-100, static_cast<int>(amax_bits >> 23) - 127);
}
__device__ __forceinline__ float pow2f(int e) {
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// Image of token t of x, one scale for the whole row: a bf16 or fp16 value keeps all its bits down
// to 2^-29 of the row's largest, and below that errs by at most 2^-40 of it.
template <class X>
__device__ void moe_convert_token(const X* x, uint8_t* xs, int t, int H, uint32_t* part) {
  const X* row = x + static_cast<int64_t>(t) * H;
  uint8_t* img = xs + t * moe_image_row(H);
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
  const int E = moe_exp(am);
  const float up = pow2f(14 - E);
  for (int c = threadIdx.x; c < H / 8; c += kMoeThreads) {
    float v[8];
    load8(row + 8 * c, v);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(v[2 * j] * up, v[2 * j + 1] * up);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(img + moe_image_offset(8 * c)) = make_uint4(w[0], w[1], w[2], w[3]);
    if ((c & 15) == 0)
      *reinterpret_cast<float*>(img + (c >> 4) * kMoeBlock + 256) = pow2f(E - 14);
  }
}

// One CTA per token, where the caller brings ids and weights.
template <class X>
__global__ void __launch_bounds__(kMoeThreads) moe_prepare_kernel(const X* x, uint8_t* xs,
                                                                 uint32_t* counters, int H) {
  __shared__ uint32_t part[kMoeWarps];
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (blockIdx.x == 0 && threadIdx.x < kMoeCounters) counters[threadIdx.x] = 0;
  moe_convert_token(x, xs, blockIdx.x, H, part);
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
  // the image of token i by CTA 7 - i, while the others may still multiply
  const int mine = kRouteCluster - 1 - static_cast<int>(rank);
  if (mine < TB && t0 + mine < p.T) moe_convert_token(x, p.xs, t0 + mine, p.H, upart);
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
  const uint8_t* s13;        // (E, 2 I, H / 16) scales: gate rows, then up rows
  const uint8_t* s2;         // (E, H, I / 16)
  const float* ts13;         // (E,)
  const float* ts2;
  const int* ids;
  const float* weights;
  const uint8_t* xs;         // images of x, one per token
  uint8_t* h;                // images of the hidden values (times weight and down scale), per pair
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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
};

// Pairs by expert. A token that names an expert twice keeps the first pair with the sum of the
// weights; ids outside [0, E) are no pair (-1 quietly, others reported). Ends with a barrier.
template <int kThreads>
__device__ void moe_plan(const MoeExpertsParams& p, MoePlan& pl) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int npairs = p.T * p.k;
  constexpr int kPer = (kMoeMaxTokens * kMoeMaxTopK + kThreads - 1) / kThreads;
  int id[kPer], pos[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int pr = tid + i * kThreads;
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
    if (id[i] >= 0) pl.pairs[pl.off[id[i]] + pos[i]] = static_cast<uint16_t>(tid + i * kThreads);
  __syncthreads();
}

// ---- the experts' kernel. Tasks of 256 weight rows of one expert, all tokens of the expert (in
// passes of 32 where more take it), K in stages of 256:
//   gate / up: 128 hidden units (128 gate rows, 128 up rows; MMA rows g: gate, g + 8: up of one
//              unit, so one thread holds both values of the same token);
//              h = silu(gate) up w ts, scaled per token by the 128 units' largest, as fp16 image;
//   down:      256 output rows of one expert and a slice of I; partial sums per (slice, pair);
//   combine:   y = the partial sums of a token's pairs in slot order.
// Warps: 16 consumers of 16 MMA rows each; a weight producer, which takes the tickets, publishes the
// tasks in a small queue and keeps the weight ring full across tasks and phases (TMA boxes of
// 128 rows x 128 bytes for the codes, cp.async for the scales, whose row pitch need not suit TMA);
// an activation producer, which copies the tokens' images (bulk copies, a lane per token) into a
// ring of two slots, waiting for the gate / up phase to end before the first hidden values.
// Bound by the weights' bytes where the tokens per expert are few: per 2048 weights a warp issues
// about 140 instructions, 35 cycles of an SM against 49 for the bytes.
constexpr int kMoeConsumers = 16;
constexpr int kMoeExpertThreads = 32 * (kMoeConsumers + 2);
constexpr int kMoeTiles = 4;                              // token tiles (8 columns) per pass
constexpr int kMoeStages = 4;
constexpr int kMoeCodes = 256 * 128;                      // codes of a stage: 256 rows, 256 of K
constexpr int kMoeStage = kMoeCodes + 256 * 16;           // and the rows' 16 scales
constexpr int kMoeActSlot = 32 * 1024;                    // activations of one chunk of K
constexpr int kMoeQueue = 4;
constexpr int oMoeAct = kMoeStages * kMoeStage;
constexpr int kMoeSmem = oMoeAct + 2 * kMoeActSlot + 1024;

struct MoeCtl {
  uint64_t wfull[kMoeStages], wempty[kMoeStages], afull[2], aempty[2], qfull[kMoeQueue],
      qempty[kMoeQueue], cbar;
  uint32_t queue[kMoeQueue];
  uint32_t abort_flag, ticket;
  uint32_t hmax[2][32];
};

// A queue entry: phase in the top two bits (0 gate / up, 1 down, 2 end), task below.
struct MoeTask {
  uint32_t phase, index;
};

// The chunks of K (in units of 128) in which nt tiles of activations are staged: as many units as a
// slot holds, an even number (a weight stage is two units).
__device__ __forceinline__ int moe_chunk_units(int nt) {
  return ((kMoeActSlot / (8 * nt) - 112) / kMoeBlock) & ~1;
}
// Bytes from token row to token row of a staged chunk of uc units: 64 mod 128, so that the 16-byte
// reads of two token rows by a lane quad each fall on different banks.
__device__ __forceinline__ uint32_t moe_pitch(int uc) {
  const uint32_t n = static_cast<uint32_t>(uc) * kMoeBlock;
  return n + ((64u - n) & 127u);
}

// Geometry of a task.
struct MoeGeom {
  int e, cnt, off;      // expert, its pairs
  int u0, u1;           // units of K
  int row0;             // first hidden unit / output row
  int z;                // slice
};
struct MoeShape {
  int blocks1, blocks2, slices;
  uint32_t total1, total2;
  __device__ __forceinline__ MoeGeom geom(const MoeExpertsParams& p, const MoePlan& pl,
                                          const MoeTask& t) const {
    MoeGeom g;
    if (t.phase == 0) {
      const int a = t.index / blocks1;
      g.e = pl.act[a];
      g.row0 = (t.index % blocks1) * 128;
      g.u0 = 0;
      g.u1 = p.H / 128;
      g.z = 0;
    } else {
      const int ab = t.index / slices;
      g.z = t.index % slices;
      g.e = pl.act[ab / blocks2];
      g.row0 = (ab % blocks2) * 256;
      const int pairs = (p.I / 128 + 1) / 2;  // slices begin on whole stages
      g.u0 = 2 * (pairs * g.z / slices);
      g.u1 = min(p.I / 128, 2 * (pairs * (g.z + 1) / slices));
    }
    g.cnt = pl.cnt[g.e];
    g.off = pl.off[g.e];
    return g;
  }
};

// One unit against NT staged token tiles. A quad reads pieces 4 (u & 1) + q of its rows' 128 bytes,
// 128B-swizzled; lane group g holds row rho(g) of its 8, rho alternating between rows 0..3 and 4..7
// so that the two rows of a read phase use different banks.
template <int NT>
__device__ __forceinline__ void moe_unit(float (&acc)[kMoeTiles][4], uint32_t codes_a,
                                         uint32_t codes_b, uint32_t scale_a, uint32_t scale_b,
                                         uint32_t tok, uint32_t tile, uint32_t fac) {
  uint32_t a[4], b[4], sa, sb;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(codes_a));
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(codes_b));
  asm volatile("ld.shared.u16 %0, [%1];" : "=r"(sa) : "r"(scale_a));
  asm volatile("ld.shared.u16 %0, [%1];" : "=r"(sb) : "r"(scale_b));
  float f[NT][2], d[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[t][0]) : "r"(fac + t * tile));
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[t][1]) : "r"(fac + t * tile + tile / 8));
#pragma unroll
    for (int c = 0; c < 4; ++c) d[t][c] = 0.0f;
  }
  const uint32_t ha = cvt_e4m3x2_f16x2(sa), hb = cvt_e4m3x2_f16x2(sb);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 xb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(xb[t].x), "=r"(xb[t].y), "=r"(xb[t].z), "=r"(xb[t].w)
                   : "r"(tok + t * tile + 64 * j));
    const uint32_t sel = j < 2 ? 0x1010 : 0x3232;
    uint32_t fa[4], fb[4];
    codes_f16(a[j], byte_perm(ha, ha, sel), fa);
    codes_f16(b[j], byte_perm(hb, hb, sel), fb);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      mma_f16(d[t], fa[0], fb[0], fa[1], fb[1], xb[t].x, xb[t].y);
      mma_f16(d[t], fa[2], fb[2], fa[3], fb[3], xb[t].z, xb[t].w);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c)  // volatile: issued before the caller releases the slot
      asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(acc[t][c]) : "f"(d[t][c]), "f"(f[t][c & 1]));
}

// A whole warp's bounded wait: the same answer in every lane.
__device__ __forceinline__ bool moe_warp_wait(uint64_t& bar, uint32_t parity, uint32_t code,
                                              MoeCtl& ctl, uint32_t* err) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&bar), parity, err, code, &ctl.abort_flag));
}

// Ring positions of a role.
struct MoeRings {
  RingPos<kMoeStages> w;
  RingPos<2> a;
  RingPos<kMoeQueue> q;
};

// A consumer warp's part of one pass: units [u0, u1) against NT tiles.
template <int NT>
__device__ __forceinline__ bool moe_consume(float (&acc)[kMoeTiles][4], const uint8_t* smem,
                                            MoeCtl& ctl, MoeRings& r, int u0, int u1, int row_a,
                                            int row_b, bool active, uint32_t* err) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int cu = moe_chunk_units(NT);
  const uint32_t base = smem_u32(smem);
  const uint32_t xa = base + row_a * 128, xb = base + row_b * 128;
  const uint32_t ya = base + kMoeCodes + row_a * 16 + 2 * q, yb = base + kMoeCodes + row_b * 16 + 2 * q;
  for (int c0 = u0; c0 < u1; c0 += cu) {
    const int uc = min(cu, u1 - c0);
    const uint32_t pitch = moe_pitch(uc);
    if (!moe_warp_wait(ctl.afull[r.a.slot], r.a.phase, kErrWaitOperand, ctl, err)) return false;
    const uint32_t act = base + oMoeAct + r.a.slot * kMoeActSlot;
    const uint32_t tok = act + g * pitch + 16 * q, fac = act + 2 * q * pitch + 256;
    for (int u = 0; u < uc; u += 2) {
      if (!moe_warp_wait(ctl.wfull[r.w.slot], r.w.phase, kErrWaitTma, ctl, err)) return false;
      const uint32_t st = r.w.slot * kMoeStage;
      if (active) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (u + v < uc)
            moe_unit<NT>(acc, xa + st + (((4 * v + q) ^ (row_a & 7)) << 4),
                         xb + st + (((4 * v + q) ^ (row_b & 7)) << 4), ya + st + 8 * v,
                         yb + st + 8 * v, tok + (u + v) * kMoeBlock, 8 * pitch,
                         fac + (u + v) * kMoeBlock);
      }
      // the MMAs that took the stage's words are issued (volatile, in order), so the loads are done
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.wempty[r.w.slot]));
      r.w.next();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&ctl.aempty[r.a.slot]));
    r.a.next();
  }
  return true;
}

// Barrier of the consumer warps: an mbarrier, so that the wait is bounded and ends when another role
// has given up.
__device__ __forceinline__ bool moe_consumer_sync(MoeCtl& ctl, uint32_t& parity, uint32_t* err) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl.cbar));
  const bool ok = moe_warp_wait(ctl.cbar, parity, kErrWaitAccum, ctl, err);
  parity ^= 1u;
  return ok;
}

// The next queue entry (lane 0 reads it, and the shuffle waits for that read before the release).
__device__ __forceinline__ bool moe_next_task(MoeTask& t, MoeCtl& ctl, MoeRings& r, uint32_t* err) {
  if (!moe_warp_wait(ctl.qfull[r.q.slot], r.q.phase, kErrWaitTma, ctl, err)) return false;
  uint32_t v = *reinterpret_cast<volatile uint32_t*>(&ctl.queue[r.q.slot]);
  v = __shfl_sync(0xFFFFFFFFu, v, 0);
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl.qempty[r.q.slot]));
  r.q.next();
  t.phase = v >> 30;
  t.index = v & 0x3FFFFFFFu;
  return true;
}

// Until *counter >= target, bounded.
__device__ __forceinline__ bool moe_wait(const uint32_t* counter, uint32_t target, MoeCtl& ctl,
                                         uint32_t* err) {
  const long long c0 = clock64();
  while (ld_acquire_gpu(counter) < target) {
    if (*reinterpret_cast<volatile uint32_t*>(&ctl.abort_flag)) return false;
    if (static_cast<unsigned long long>(clock64() - c0) > kWaitLimitCycles) {
      atomicOr(err, kErrWaitOperand);
      *reinterpret_cast<volatile uint32_t*>(&ctl.abort_flag) = 1u;
      return false;
    }
  }
  return true;
}

__global__ void __launch_bounds__(kMoeExpertThreads, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap tm_w13,
                       const __grid_constant__ CUtensorMap tm_w2, const MoeExpertsParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ MoePlan pl;
  __shared__ MoeCtl ctl;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    ctl.abort_flag = 0;
    for (int s = 0; s < kMoeStages; ++s) {
      mbar_init(smem_u32(&ctl.wfull[s]), 33);  // the tx arrive and 32 lanes' scale copies
      mbar_init(smem_u32(&ctl.wempty[s]), kMoeConsumers);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&ctl.afull[s]), 1);
      mbar_init(smem_u32(&ctl.aempty[s]), kMoeConsumers);
    }
    for (int s = 0; s < kMoeQueue; ++s) {
      mbar_init(smem_u32(&ctl.qfull[s]), 1);
      mbar_init(smem_u32(&ctl.qempty[s]), kMoeConsumers + 1);
    }
    mbar_init(smem_u32(&ctl.cbar), kMoeConsumers);
    fence_mbar_init();
  }
  if (tid < 64) ctl.hmax[tid >> 5][tid & 31] = 0;
  for (int e = tid; e < p.E; e += kMoeExpertThreads) pl.cnt[e] = 0;
  __syncthreads();
  grid_dep_wait();
  moe_plan<kMoeExpertThreads>(p, pl);
  const int nact = pl.nact;

  MoeShape sh;
  sh.blocks1 = p.I / 128;
  sh.total1 = static_cast<uint32_t>(nact) * sh.blocks1;
  sh.blocks2 = (p.H + 255) / 256;
  // slices of I per down task: while the tasks do not fill the grid and the partials fit
  sh.slices = 1;
  while (nact * sh.blocks2 * sh.slices < static_cast<int>(gridDim.x) &&
         2 * sh.slices * p.T * p.k <= p.part_rows && p.I / 128 >= 4 * sh.slices)
    sh.slices *= 2;
  sh.total2 = static_cast<uint32_t>(nact) * sh.blocks2 * sh.slices;

  MoeRings r;
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  if (warp == kMoeConsumers) {
    // ------------------------------------------------------------------ weight producer
    if (lane == 0) {
      prefetch_tmap(&tm_w13);
      prefetch_tmap(&tm_w2);
    }
    uint32_t phase = 0;
    int issued = 0;
    while (true) {
      // the next task: the phase's tickets, then the next phase's
      MoeTask t{2, 0};
      while (phase < 2) {
        uint32_t k = 0;
        if (lane == 0) k = atomicAdd(p.counters + (phase == 0 ? kMoeGateUp : kMoeDown), 1u);
        k = __shfl_sync(0xFFFFFFFFu, k, 0);
        if (k < (phase == 0 ? sh.total1 : sh.total2)) {
          t.phase = phase;
          t.index = k;
          break;
        }
        ++phase;
      }
      if (!moe_warp_wait(ctl.qempty[r.q.slot], r.q.phase ^ 1u, kErrWaitEmpty, ctl, p.err)) break;
      if (lane == 0) {
        ctl.queue[r.q.slot] = t.phase << 30 | t.index;
        mbar_arrive(smem_u32(&ctl.qfull[r.q.slot]));
      }
      r.q.next();
      if (t.phase == 2) break;
      const MoeGeom gm = sh.geom(p, pl, t);
      const bool up = t.phase == 0;
      const int K = up ? p.H : p.I;
      const uint8_t* sc = up ? p.s13 : p.s2;
      // rows 0..127 and 128..255 of the tile
      const int64_t ra = up ? static_cast<int64_t>(gm.e) * 2 * p.I + gm.row0
                            : static_cast<int64_t>(gm.e) * p.H + gm.row0;
      const int64_t rb = up ? ra + p.I : ra + 128;
      const bool two = up || gm.row0 + 128 < p.H;
      bool ok = true;
      for (int c0 = 0; c0 < gm.cnt && ok; c0 += 8 * kMoeTiles) {
        for (int u = gm.u0; u < gm.u1; u += 2) {
          if (!moe_warp_wait(ctl.wempty[r.w.slot], r.w.phase ^ 1u, kErrWaitEmpty, ctl, p.err)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + r.w.slot * kMoeStage;
          const uint32_t fb = smem_u32(&ctl.wfull[r.w.slot]);
          if (lane == 0) {
            const CUtensorMap* tm = up ? &tm_w13 : &tm_w2;
            mbar_arrive_expect_tx(fb, two ? kMoeCodes : kMoeCodes / 2);
            tma_load_2d(smem_u32(st), tm, u * 64, static_cast<int32_t>(ra), fb);
            if (two)
              tma_load_2d(smem_u32(st + kMoeCodes / 2), tm, u * 64, static_cast<int32_t>(rb), fb);
          }
          const bool second = u + 1 < gm.u1;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = lane + 32 * i;
            if (i >= 4 && !two) break;
            const uint8_t* src = sc + ((i < 4 ? ra : rb) + (row & 127)) * (K / 16) + u * 8;
            const uint32_t dst = smem_u32(st + kMoeCodes + row * 16);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
            if (second)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + 8), "l"(src + 8)
                           : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(fb) : "memory");
          r.w.next();
          ++issued;
        }
      }
      if (!ok) break;
    }
    // every copy issued has landed before the CTA exits (also after a wait ran out)
    for (int j = max(0, issued - kMoeStages); j < issued; ++j)
      mbar_wait(smem_u32(&ctl.wfull[j % kMoeStages]), (j / kMoeStages) & 1, p.err, kErrWaitTma,
                nullptr);
  } else if (warp == kMoeConsumers + 1) {
    // -------------------------------------------------------------- activation producer
    bool ready = false;
    int issued = 0;
    MoeTask t;
    while (moe_next_task(t, ctl, r, p.err) && t.phase != 2) {
      if (t.phase == 1 && !ready) {
        if (!__all_sync(0xFFFFFFFFu,
                        moe_wait(p.counters + kMoeGateUpDone, sh.total1, ctl, p.err)))
          break;
        // the hidden values were written by ordinary stores; the copies read through the async proxy
        asm volatile("fence.proxy.async;" ::: "memory");
        ready = true;
      }
      const MoeGeom gm = sh.geom(p, pl, t);
      bool ok = true;
      for (int c0 = 0; c0 < gm.cnt && ok; c0 += 8 * kMoeTiles) {
        const int n = min(gm.cnt - c0, 8 * kMoeTiles), nt = (n + 7) / 8;
        const int cu = moe_chunk_units(nt);
        const uint8_t* src = nullptr;
        if (lane < n) {
          const int pr = pl.pairs[gm.off + c0 + lane];
          src = t.phase == 0 ? p.xs + (pr / p.k) * moe_image_row(p.H)
                             : p.h + pr * moe_image_row(p.I);
        }
        for (int u = gm.u0; u < gm.u1; u += cu) {
          const int uc = min(cu, gm.u1 - u);
          if (!moe_warp_wait(ctl.aempty[r.a.slot], r.a.phase ^ 1u, kErrWaitEmpty, ctl, p.err)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&ctl.afull[r.a.slot]);
          if (lane == 0) mbar_arrive_expect_tx(fb, static_cast<uint32_t>(n * uc) * kMoeBlock);
          __syncwarp();
          if (lane < n)
            bulk_load(smem_u32(smem + oMoeAct + r.a.slot * kMoeActSlot) + lane * moe_pitch(uc),
                      src + static_cast<int64_t>(u) * kMoeBlock, uc * kMoeBlock, fb);
          r.a.next();
          ++issued;
        }
      }
      if (!ok) break;
    }
    for (int j = max(0, issued - 2); j < issued; ++j)
      mbar_wait(smem_u32(&ctl.afull[j % 2]), (j / 2) & 1, p.err, kErrWaitTma, nullptr);
  } else {
    // ---------------------------------------------------------------------------- consumers
    const int g = lane >> 2, q = lane & 3;
    const int rho = (g >> 1) | ((g & 1) << 2);
    int flip = 0;
    uint32_t cph = 0;
    bool ok = true;
    MoeTask t;
    // any wait that runs out ends the role (ok false): the abort flag ends the other roles' waits
    while ((ok = moe_next_task(t, ctl, r, p.err)) && t.phase != 2) {
      const MoeGeom gm = sh.geom(p, pl, t);
      const bool up = t.phase == 0;
      const int row_a = up ? 8 * warp + rho : 16 * warp + rho;
      const int row_b = up ? row_a + 128 : row_a + 8;
      const bool active = up || gm.row0 + 16 * warp < p.H;
      for (int c0 = 0; c0 < gm.cnt && ok; c0 += 8 * kMoeTiles) {
        const int n = min(gm.cnt - c0, 8 * kMoeTiles), nt = (n + 7) / 8;
        float acc[kMoeTiles][4] = {};
        if (nt == 1) ok = moe_consume<1>(acc, smem, ctl, r, gm.u0, gm.u1, row_a, row_b, active, p.err);
        else if (nt == 2) ok = moe_consume<2>(acc, smem, ctl, r, gm.u0, gm.u1, row_a, row_b, active, p.err);
        else if (nt == 3) ok = moe_consume<3>(acc, smem, ctl, r, gm.u0, gm.u1, row_a, row_b, active, p.err);
        else ok = moe_consume<4>(acc, smem, ctl, r, gm.u0, gm.u1, row_a, row_b, active, p.err);
        if (!ok) break;
        if (up) {
          const float ts13 = p.ts13[gm.e], ts2 = p.ts2[gm.e];
          const int i = gm.row0 + 8 * warp + rho;
#pragma unroll
          for (int tl = 0; tl < kMoeTiles; ++tl) {
            if (tl >= nt) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int col = 8 * tl + 2 * q + c;
              float hv = 0.0f;
              if (col < n)
                hv = silu_rn(acc[tl][c] * ts13) * (acc[tl][2 + c] * ts13) *
                     (pl.w[pl.pairs[gm.off + c0 + col]] * ts2);
              acc[tl][c] = hv;
              uint32_t hm = __float_as_uint(hv) & 0x7FFFFFFFu;
              hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, 4));
              hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, 8));
              hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, 16));
              if (g == 0 && col < n) atomicMax(&ctl.hmax[flip][col], hm);
            }
          }
          if (!(ok = moe_consumer_sync(ctl, cph, p.err))) break;
          if (tid < 32) ctl.hmax[flip ^ 1][tid] = 0;
#pragma unroll
          for (int tl = 0; tl < kMoeTiles; ++tl) {
            if (tl >= nt) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int col = 8 * tl + 2 * q + c;
              if (col < n) {
                const int E = moe_exp(ctl.hmax[flip][col]);
                uint8_t* img = p.h + pl.pairs[gm.off + c0 + col] * moe_image_row(p.I);
                *reinterpret_cast<__half*>(img + moe_image_offset(i)) =
                    __float2half_rn(acc[tl][c] * pow2f(14 - E));
                if (warp == 0 && g == 0)
                  *reinterpret_cast<float*>(img + gm.row0 / 128 * kMoeBlock + 256) = pow2f(E - 14);
              }
            }
          }
          flip ^= 1;
          // hmax is read, the other copy cleared, the images written
          if (!(ok = moe_consumer_sync(ctl, cph, p.err))) break;
        } else if (active) {
#pragma unroll
          for (int tl = 0; tl < kMoeTiles; ++tl) {
            if (tl >= nt) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int col = 8 * tl + 2 * q + c;
              if (col < n) {
                const int pr = pl.pairs[gm.off + c0 + col];
                float* dst = p.part + (static_cast<int64_t>(gm.z) * p.T * p.k + pr) * p.H + gm.row0;
                dst[row_a] = acc[tl][c];
                dst[row_b] = acc[tl][2 + c];
              }
            }
          }
        }
      }
      if (!ok || (!up && !(ok = moe_consumer_sync(ctl, cph, p.err)))) break;
      if (tid == 0) {
        if (up) asm volatile("fence.proxy.async;" ::: "memory");
        __threadfence();
        atomicAdd(p.counters + (up ? kMoeGateUpDone : kMoeDownDone), 1u);
      }
    }

    // ------------------------------------------------------------------------------ combine
    const int cols = 4 * 32 * kMoeConsumers;  // outputs per task
    const int blocks3 = (p.H + cols - 1) / cols;
    bool ready = false;
    while (ok) {
      if (!moe_consumer_sync(ctl, cph, p.err)) break;
      if (tid == 0) {
        ctl.ticket = atomicAdd(p.counters + kMoeCombine, 1u);
        if (!ready && ctl.ticket < static_cast<uint32_t>(p.T * blocks3))
          moe_wait(p.counters + kMoeDownDone, sh.total2, ctl, p.err);  // raises the abort flag
      }
      if (!moe_consumer_sync(ctl, cph, p.err) || *abort_flag) break;
      const uint32_t task = ctl.ticket;
      if (task >= static_cast<uint32_t>(p.T * blocks3)) break;
      ready = true;
      const int t = task / blocks3, h0 = (task % blocks3) * cols + 4 * tid;
      if (h0 >= p.H) continue;
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int s = 0; s < p.k; ++s) {
        const int pr = t * p.k + s;
        if (!pl.used[pr]) continue;
        for (int z = 0; z < sh.slices; ++z) {
          const uint4 v = ld_cg(p.part + (static_cast<int64_t>(z) * p.T * p.k + pr) * p.H + h0);
          o[0] += __uint_as_float(v.x);
          o[1] += __uint_as_float(v.y);
          o[2] += __uint_as_float(v.z);
          o[3] += __uint_as_float(v.w);
        }
      }
      store_row<4>(p.y, static_cast<int64_t>(t) * p.H + h0, o, p.out_dtype, p.vec_out);
    }
  }
}

}  // namespace bd
