// gemm_fp4.cuh -- W4A4 GEMM for sm_100a: C = A4 . B4^T with both operands in microscaled 4-bit
// floating point (NVFP4 or MXFP4), consumed by tcgen05.mma kind::mxf4nvf4 / kind::mxf4 as they
// are: no transcode, codes and scale tiles go from HBM to shared memory by TMA / bulk copies,
// scales on to tensor memory by tcgen05.cp.
//
//   C[m, n] = act(acc[m, n] * ((s_m * ts) * s_n) + bias[n]),  acc = sum_k a b in fp32
//
// Two kernels: w4a4_pair_kernel where 256 x 256 tiles fill the machine, w4a4_gemm_kernel else.
//
// w4a4_gemm_kernel: tiles of 128 weight rows (the MMA's M) x BN tokens (its N), so a decode batch
// of 16 tokens pads to 16 columns instead of 128 rows. One CTA computes one K slice of one tile;
// the `split` CTAs of a cluster share a tile, and exchange their fp32 partials through distributed
// shared memory, each summing its share of the columns in rank order: no workspace, no atomics,
// the same bits whatever the timing.
//
// Warps: 0 producer (TMA), 1 MMA, all four drain the accumulator (lane = weight row).
//
// Bound by latency and, where there are weights enough, their bytes. Measured with the quantiser in
// front, one call after another on weights that are not in L2: 1 token, 4096 -> 14336 (33 MB) 12 us, 2.7
// TB/s; 32 tokens, 14336 -> 4096 (31 MB) 14 to 18 us; 128 tokens, 4096 -> 4096 12 us; 333 tokens, 1056 ->
// 1000 18 us.
#pragma once
#include <cstdint>

#include "epilogue.cuh"
#include "fp4.cuh"
#include "sm100.cuh"

namespace bd {

struct GemmFp4Params {
  void* out;
  const uint8_t* sf_t;        // scale tiles of the tokens / of the weights
  const uint8_t* sf_w;
  const float* row_scale_t;   // per token row / per weight row, may be null
  const float* row_scale_w;
  const __nv_bfloat16* bias;
  float tensor_scale;
  int M, N, K, words;
  int n_tiles, m_tiles;
  int out_dtype, epilogue;
  int vec_out;                // rows of C are 16-byte aligned
  int weights_early;
  uint32_t* err;
};

constexpr int kF4ChunkK = 256;  // elements of K per stage: 128 bytes of codes, a swizzle row

constexpr int cround_up(int x, int a) { return (x + a - 1) / a * a; }

template <int BN, int kFmt>
struct GemmFp4Cfg {
  static constexpr int kWords = kFmt == kNvfp4 ? 4 : 2;  // scale words per row and chunk
  static constexpr int kWBytes = 128 * 128;              // weight codes of a stage
  static constexpr int kTBytes = BN * 128;               // token codes
  static constexpr int kSfBytes = 512 * kWords;          // scales of 128 rows
  static constexpr int oT = kWBytes;
  static constexpr int oSw = oT + kTBytes;
  static constexpr int oSt = oSw + kSfBytes;
  static constexpr int kStage = cround_up(oSt + kSfBytes, 1024);
  // two CTAs per SM up to 64 tokens (weight streaming: twice the independent schedules), one above
  static constexpr int kCtasPerSm = BN <= 64 ? 2 : 1;
  static constexpr int kBudget = (kCtasPerSm == 2 ? 113 : 226) * 1024 - 2048 - 1024;
  static constexpr int kStages = kBudget / kStage > 8 ? 8 : kBudget / kStage;
  static constexpr int kRing = kStages * kStage;
  // partial exchange: [split][BN / split / 2][128][2] fp32, over the ring
  static_assert(BN * 128 * 4 <= kRing, "exchange buffer fits the ring");
  static constexpr int kSmemBytes = kRing + 2048 + 1024;
  // tensor memory: accumulator, then two sets of scale words
  static constexpr int kSfSet = 4 * kWords * 2;
  static constexpr int kSfCol0 = BN < 64 ? 64 : BN;
  static constexpr int kUsedCols = kSfCol0 + 2 * kSfSet;
  static constexpr int kTmemCols = kUsedCols <= 128 ? 128 : kUsedCols <= 256 ? 256 : 512;
  static_assert(kUsedCols <= 512, "tensor memory budget");
  static_assert(BN % 16 == 0 && BN <= 128, "MMA N");
  static_assert(kStage % 1024 == 0 && kWBytes % 1024 == 0 && kTBytes % 1024 == 0,
                "1 KB swizzle atoms");
};

struct GemmFp4Ctl {
  uint64_t full[8], empty[8], done;
  uint32_t tmem_base, abort_flag;
  uint32_t peer_failed;  // set by a CTA of the cluster whose partial is not there
  float tok_scale[128];
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CTAs of a cluster that add one another's partials: between the barrier after which partials are written
// and the one after which they are read, a CTA without one (a wait ran out) says so to all; `failed` (zero
// before the first barrier) is then set in every CTA after the second.
__device__ __forceinline__ void cluster_report_failure(uint32_t* failed, int ctas) {
  if (static_cast<int>(threadIdx.x) < ctas)
    st_shared_cluster_u32(mapa_shared(smem_u32(failed), threadIdx.x), 1u);
  __syncwarp();
}

__device__ __forceinline__ float activate(float v, int epi) {
  if (epi == 2) return fmaxf(v, 0.0f);
  if (epi == 3) return silu_rn(v);
  if (epi == 4) return gelu_tanh_rn(v);
  return v;
}

template <int BN, int kFmt>
__global__ void __launch_bounds__(128, (GemmFp4Cfg<BN, kFmt>::kCtasPerSm))
    w4a4_gemm_kernel(const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_t, const GemmFp4Params p, int split) {
  using Cfg = GemmFp4Cfg<BN, kFmt>;
  constexpr bool kNv = kFmt == kNvfp4;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  GemmFp4Ctl& ctl = *reinterpret_cast<GemmFp4Ctl*>(smem + Cfg::kRing);
  static_assert(sizeof(GemmFp4Ctl) <= 2048, "control block");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abort_flag = &ctl.abort_flag;

  const int tile = blockIdx.x / split, rank = blockIdx.x % split;
  const int mt = tile % p.m_tiles, nt = tile / p.m_tiles;
  const int n0 = nt * 128, m0 = mt * BN;
  const int chunks = (p.K + kF4ChunkK - 1) / kF4ChunkK;
  const int k0 = static_cast<int>(static_cast<int64_t>(chunks) * rank / split);
  const int k1 = static_cast<int>(static_cast<int64_t>(chunks) * (rank + 1) / split);

  if (tid == 0) {
    ctl.abort_flag = 0;
    ctl.peer_failed = 0;
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(smem_u32(&ctl.full[s]), 1);
      mbar_init(smem_u32(&ctl.empty[s]), 1);
    }
    mbar_init(smem_u32(&ctl.done), 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctl.tmem_base), Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = ctl.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&tm_w);
      prefetch_tmap(&tm_t);
      // words of chunk k present in the tiles
      auto words_of = [&](int k) { return min(Cfg::kWords, p.words - k * Cfg::kWords); };
      auto load_weights = [&](int k, int slot) {
        uint8_t* st = smem + slot * Cfg::kStage;
        const uint32_t fb = smem_u32(&ctl.full[slot]);
        const uint32_t sfb = 512u * words_of(k);
        mbar_arrive_expect_tx(fb, Cfg::kWBytes + Cfg::kTBytes + 2 * sfb);
        tma_load_2d(smem_u32(st), &tm_w, k * 128, n0, fb);
        bulk_load(smem_u32(st + Cfg::oSw),
                  p.sf_w + (static_cast<int64_t>(nt) * p.words + k * Cfg::kWords) * 512, sfb, fb);
      };
      auto load_tokens = [&](int k, int slot) {
        uint8_t* st = smem + slot * Cfg::kStage;
        const uint32_t fb = smem_u32(&ctl.full[slot]);
        const uint32_t sfb = 512u * words_of(k);
        tma_load_2d(smem_u32(st + Cfg::oT), &tm_t, k * 128, m0, fb);
        bulk_load(smem_u32(st + Cfg::oSt),
                  p.sf_t + (static_cast<int64_t>(m0 / 128) * p.words + k * Cfg::kWords) * 512, sfb, fb);
      };
      // the first ring of weights before the wait for the previous grid (when it does not write
      // them), the tokens after it
      const int first = min(k1 - k0, Cfg::kStages);
      if (!p.weights_early) grid_dep_wait();
      for (int i = 0; i < first; ++i) load_weights(k0 + i, i);
      grid_dep_wait();
      // only now: the next grid may load weights that the grid before this one wrote
      grid_dep_launch_dependents();
      for (int i = 0; i < first; ++i) load_tokens(k0 + i, i);
      RingPos<Cfg::kStages> r;
      for (int i = 0; i < first; ++i) r.next();
      for (int k = k0 + first; k < k1; ++k) {
        if (!mbar_wait(smem_u32(&ctl.empty[r.slot]), r.phase ^ 1u, p.err, kErrWaitEmpty,
                       abort_flag))
          break;
        load_weights(k, r.slot);
        load_tokens(k, r.slot);
        r.next();
      }
      // a wait ran out: what was issued last to each slot lands before the CTA goes on
      for (int s = 0; s < Cfg::kStages && *abort_flag; ++s)
        mbar_wait(smem_u32(&ctl.full[s]), r.last_parity(s), p.err, kErrWaitTma, nullptr,
                  kWaitLimitCycles / 8);
    }
  } else if (warp == 1) {
    RingPos<Cfg::kStages> r;
    for (int k = k0; k < k1; ++k) {
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl.full[r.slot]), r.phase, p.err,
                                             kErrWaitTma, abort_flag)))
        break;
      tc_fence_after();
      const uint32_t st = smem_u32(smem + r.slot * Cfg::kStage);
      const uint32_t sfw = tb + Cfg::kSfCol0 + ((k - k0) & 1) * Cfg::kSfSet;
      const uint32_t sft = sfw + 4 * Cfg::kWords;
      const int words = min(Cfg::kWords, p.words - k * Cfg::kWords);
      const int steps = min(4, (p.K - k * kF4ChunkK + 63) / 64);
      if (elect_one()) {
        for (int w = 0; w < words; ++w) {
          tmem_cp_32x128b_x4(sfw + 4 * w, sdesc_sf(st + Cfg::oSw + 512 * w));
          tmem_cp_32x128b_x4(sft + 4 * w, sdesc_sf(st + Cfg::oSt + 512 * w));
        }
        for (int kk = 0; kk < steps; ++kk) {
          const int w = kNv ? kk : kk >> 1;
          const uint32_t idesc = idesc_mxf4(128, BN, !kNv, kNv ? 0 : 2 * (kk & 1));
          mma_mxf4_ss<kNv, false>(tb, sdesc_sw128(st + kk * 32), sdesc_sw128(st + Cfg::oT + kk * 32),
                                  idesc, sfw + 4 * w, sft + 4 * w,
                                  (k > k0 || kk > 0) ? 1u : 0u);
        }
        tc_commit(smem_u32(&ctl.empty[r.slot]));
      }
      __syncwarp();
      r.next();
    }
    if (elect_one()) tc_commit(smem_u32(&ctl.done));
    __syncwarp();
  }
  __syncwarp();
  // ---- drain: every thread owns weight row n0 + 32 warp + lane of the tile
  grid_dep_wait();
  for (int j = tid; j < BN; j += 128) {
    const int m = m0 + j;
    ctl.tok_scale[j] = p.row_scale_t != nullptr && m < p.M
                           ? __fmul_rn(p.row_scale_t[m], p.tensor_scale)
                           : p.tensor_scale;
  }
  const int n = n0 + 32 * warp + lane;
  const float wscale = p.row_scale_w != nullptr && n < p.N ? p.row_scale_w[n] : 1.0f;
  const float bias = p.epilogue != 0 && n < p.N ? __bfloat162float(p.bias[n]) : 0.0f;
  bool ok = mbar_wait(smem_u32(&ctl.done), 0, p.err, kErrWaitAccum, abort_flag);
  // the barrier publishes tok_scale; nothing is stored after a wait that ran out, here or in a peer of
  // the cluster
  ok = __syncthreads_and(ok) && !*abort_flag;
  tc_fence_after();
  const uint32_t taddr = tb + (static_cast<uint32_t>(32 * warp) << 16);
  // NC finished columns j .. of this thread's weight row: a warp's stores of a column are side by side
  auto finish = [&](int j, auto& acc) {
    constexpr int NC = sizeof(acc) / sizeof(acc[0]);
    float v[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] = __fmul_rn(acc[i], ctl.tok_scale[j + i]);
    if (p.row_scale_w != nullptr) {
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = __fmul_rn(v[i], wscale);
    }
    if (p.epilogue != 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = activate(__fadd_rn(v[i], bias), p.epilogue);
    }
    const int cols = min(NC, p.M - m0 - j);
    if (n >= p.N) return;
    const int64_t at = static_cast<int64_t>(m0 + j) * p.N + n;
    auto store = [&](auto* out, auto convert) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (i < cols) out[at + static_cast<int64_t>(i) * p.N] = convert(v[i]);
    };
    if (p.out_dtype == 0)
      store(static_cast<__nv_bfloat16*>(p.out), [](float x) { return __float2bfloat16_rn(x); });
    else if (p.out_dtype == 1)
      store(static_cast<__half*>(p.out), [](float x) { return __float2half_rn(x); });
    else store(static_cast<float*>(p.out), [](float x) { return x; });
  };
  if (split == 1) {
    if (ok) {
      const int cols = min(BN, p.M - m0);
#pragma unroll 1
      for (int c0 = 0; c0 < cols; c0 += 16) {
        uint32_t r[16];
        tmem_ld_x16(taddr + c0, r);
        tmem_ld_wait_x16(r);
        float acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = __uint_as_float(r[j]);
        finish(c0, acc);
      }
    }
  } else {
    // every CTA of the cluster is past its last MMA: the rings may be overwritten
    cluster_arrive();
    cluster_wait();
    // partials to the owner of the columns, pairs of columns side by side: [rank][pair][row][2]
    const int width = BN / split;  // columns per rank, at least two
    const uint32_t part = smem_u32(smem);
    const int row = 32 * warp + lane;
    if (!ok) cluster_report_failure(&ctl.peer_failed, split);
#pragma unroll 1
    for (int c0 = 0; ok && c0 < BN; c0 += 16) {
      uint32_t r[16];
      tmem_ld_x16(taddr + c0, r);
      tmem_ld_wait_x16(r);
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const int owner = (c0 + j) / width, pair = ((c0 + j) % width) / 2;
        const uint32_t at = part + ((rank * (width / 2) + pair) * 128 + row) * 8;
        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(mapa_shared(at, owner)),
                     "r"(r[j]), "r"(r[j + 1])
                     : "memory");
      }
    }
    cluster_arrive();
    cluster_wait();
    ok = *reinterpret_cast<volatile uint32_t*>(&ctl.peer_failed) == 0;
    // columns 2 pair .. of this rank: the partials in rank order, four pairs at a time where there are
    // as many (one pair's epilogue is a chain of dependent steps, and a warp has its scheduler alone)
    auto join = [&](int pair, auto& acc) {
      constexpr int NP = sizeof(acc) / sizeof(acc[0]) / 2;
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < split) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float2 v = *reinterpret_cast<const float2*>(
                smem + ((s * (width / 2) + pair + i) * 128 + row) * 8);
            acc[2 * i] = s ? acc[2 * i] + v.x : v.x;
            acc[2 * i + 1] = s ? acc[2 * i + 1] + v.y : v.y;
          }
        }
      finish(rank * width + 2 * pair, acc);
    };
    if (ok && width % 8 == 0) {
#pragma unroll 1
      for (int pair = 0; pair < width / 2; pair += 4) {
        float acc[8];
        join(pair, acc);
      }
    } else if (ok) {
      for (int pair = 0; pair < width / 2; ++pair) {
        float acc[2];
        join(pair, acc);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tb, Cfg::kTmemCols);
  }
}

// Diagnostic of the exchange above: a cluster whose CTA `failing` waits for an arrival that never comes, with
// a limit of `limit` cycles; every CTA writes whether it would store.
__global__ void __launch_bounds__(128) cluster_wait_selftest_kernel(uint32_t* stored, int ctas, int failing,
                                                                    unsigned long long limit, uint32_t* err) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ uint32_t failed;
  const int rank = static_cast<int>(cluster_ctarank());
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    failed = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const bool ok = rank != failing || mbar_wait(smem_u32(&bar), 0, err, kErrWaitAccum, nullptr, limit);
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (!ok) cluster_report_failure(&failed, ctas);
  cluster_arrive();
  cluster_wait();
  if (threadIdx.x == 0) stored[rank] = *reinterpret_cast<volatile uint32_t*>(&failed) == 0 ? 1u : 0u;
}

// w4a4_pair_kernel: tiles of 256 tokens x 256 weight rows on clusters of two CTAs (cta_group::2): CTA
// rank r loads tokens 128 r .. and weight rows 128 r .. of the tile (and the scales of all 256 weight
// rows), each stage 38 KB for 512 cycles of MMA; rank 0 issues the MMAs. Persistent, tiles dealt
// round-robin over the clusters, tokens fastest.
//
// Tensor memory: one 256-column accumulator and two sets of scale words (a second accumulator would
// leave no room for scales), so the next tile's MMAs wait for the drain: eight epilogue warps take a
// tile's 128 columns each into 128 registers in one go and release the accumulator before they scale,
// convert and store (about 300 cycles of a 4096-deep tile's 8200).
//
// Measured: 8192 x 14336 x 4096 NVFP4 213 us (4.5 PFLOP/s, the tensor pipe 58 % busy), 8192 x 4096 x
// 14336 MXFP4 183 us (5.3 PFLOP/s, 68 %). The scale copies share the tensor core with the MMAs, but
// little of the rest is theirs: without any, NVFP4 took 5 % less and MXFP4 the same.
//
// Both CTAs' loads complete on rank 0's barrier (a relay warp in rank 1 that passed arrivals on was
// 840 cycles a stage).
//
// A lane of the epilogue owns a token's row. Rows of C that do not start on 16 bytes (N * size % 16) are
// stored element by element, 32 rows at a time: 4096 x 1333 x 1024 to bf16 81 us, 4096 x 1336 x 1024 15.
// Bias and activation are not hidden behind the next tile's MMAs (the accumulator is), and show where K is
// short: 4096 x 4096 x 1024 20 us, with bias 26, GELU 44, SiLU 56; 8192 x 14336 x 4096 217, 229, 303, 395.
//
// Warps: 0 producer, 1 MMA (rank 0), 2 and 3 idle, 4..11 epilogue.
constexpr int kPairThreads = 384;

template <int kFmt>
struct PairFp4Cfg {
  static constexpr int kWords = kFmt == kNvfp4 ? 4 : 2;
  static constexpr int kCodes = 128 * 128;        // codes of 128 rows, 256 of K
  static constexpr int kSf = 512 * kWords;        // scales of 128 rows
  static constexpr int oW = kCodes;               // tokens first
  static constexpr int oSt = 2 * kCodes;
  static constexpr int oSw = oSt + kSf;           // two blocks of 128 weight rows
  static constexpr int kStage = cround_up(oSw + 2 * kSf, 1024);
  static constexpr int kStages = 5;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kSfSet = 12 * kWords;      // scale words of a stage in tensor memory
  static constexpr int kBatch = 2;                // stages whose scales are copied at once
  static constexpr int kSfCol0 = 256;
  static_assert(kSfCol0 + 2 * kBatch * kSfSet <= 512, "tensor memory budget");
  static_assert(kStage % 1024 == 0, "1 KB swizzle atoms");
};

struct PairFp4Ctl {
  uint64_t full[5], empty[5], acc_full, acc_empty, drain;
  uint32_t tmem_base, abort_flag;
};

template <int kFmt>
__global__ void __launch_bounds__(kPairThreads, 1)
    w4a4_pair_kernel(const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_t,
                     const __grid_constant__ CUtensorMap tm_sw,
                     const __grid_constant__ CUtensorMap tm_st, const GemmFp4Params p) {
  using Cfg = PairFp4Cfg<kFmt>;
  constexpr bool kNv = kFmt == kNvfp4;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ PairFp4Ctl ctl;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster = blockIdx.x / 2, clusters = gridDim.x / 2;
  const int tiles = p.n_tiles * p.m_tiles;
  const int chunks = (p.K + kF4ChunkK - 1) / kF4ChunkK;
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  if (tid == 0) {
    ctl.abort_flag = 0;
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(smem_u32(&ctl.full[s]), 1);
      mbar_init(smem_u32(&ctl.empty[s]), 1);
    }
    mbar_init(smem_u32(&ctl.acc_full), 1);
    mbar_init(smem_u32(&ctl.acc_empty), 16);  // the epilogue warps of both CTAs
    mbar_init(smem_u32(&ctl.drain), 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctl.tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before anyone arrives
  tc_fence_after();
  const uint32_t tb = ctl.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&tm_w);
      prefetch_tmap(&tm_t);
      prefetch_tmap(&tm_sw);
      prefetch_tmap(&tm_st);
      grid_dep_wait();
      grid_dep_launch_dependents();
      RingPos<Cfg::kStages> r;
      int issued = 0;
      bool ok = true;
      for (int tile = cluster; tile < tiles && ok; tile += clusters) {
        const int m0 = tile % p.m_tiles * 256 + 128 * static_cast<int>(rank);
        const int n0 = tile / p.m_tiles * 256;
        for (int k = 0; k < chunks; ++k) {
          if (!(ok = mbar_wait(smem_u32(&ctl.empty[r.slot]), r.phase ^ 1u, p.err, kErrWaitEmpty,
                               abort_flag)))
            break;
          const uint32_t st = smem_u32(smem + r.slot * Cfg::kStage);
          const uint32_t fb = mapa_shared(smem_u32(&ctl.full[r.slot]), 0);
          if (rank == 0)
            mbar_arrive_expect_tx(smem_u32(&ctl.full[r.slot]), 2 * (2 * Cfg::kCodes + 3 * Cfg::kSf));
          tma_load_2d_pair(st, &tm_t, k * 128, m0, fb);
          tma_load_2d_pair(st + Cfg::oW, &tm_w, k * 128, n0 + 128 * static_cast<int>(rank), fb);
          // scale boxes of kWords words: past a row's last word they take words of the next 128 rows
          // (or zeros), which no MMA reads
          const int w0 = k * Cfg::kWords;
          tma_load_2d_pair(st + Cfg::oSt, &tm_st, 0, m0 / 128 * p.words + w0, fb);
          tma_load_2d_pair(st + Cfg::oSw, &tm_sw, 0, n0 / 128 * p.words + w0, fb);
          tma_load_2d_pair(st + Cfg::oSw + Cfg::kSf, &tm_sw, 0, (n0 / 128 + 1) * p.words + w0, fb);
          r.next();
          ++issued;
        }
      }
      // a wait ran out: every copy issued lands before the CTA exits (rank 0's barriers say so)
      if (*abort_flag && rank == 0)
        for (int j = max(0, issued - Cfg::kStages); j < issued; ++j)
          mbar_wait(smem_u32(&ctl.full[j % Cfg::kStages]), (j / Cfg::kStages) & 1, p.err, kErrWaitTma,
                    nullptr);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      RingPos<Cfg::kStages> r;
      uint32_t aph = 0, set = 0;
      bool ok = true;
      for (int tile = cluster; tile < tiles && ok; tile += clusters) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait<true>(smem_u32(&ctl.acc_empty), aph ^ 1u, p.err,
                                                           kErrWaitAccum, abort_flag))))
          break;
        aph ^= 1u;
        tc_fence_after();
        // kBatch stages at a time: their scale copies, then their MMAs. Every change between copies
        // and MMAs costs the tensor core about 100 cycles (copies issued between the MMAs of the
        // stage before took 1.6 times as long).
        for (int k0 = 0; k0 < chunks && ok; k0 += Cfg::kBatch) {
          uint32_t st[Cfg::kBatch], free[Cfg::kBatch];
#pragma unroll
          for (int b = 0; b < Cfg::kBatch; ++b) {
            if (k0 + b >= chunks) break;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait<true>(smem_u32(&ctl.full[r.slot]), r.phase,
                                                               p.err, kErrWaitTma, abort_flag))))
              break;
            st[b] = smem_u32(smem + r.slot * Cfg::kStage);
            free[b] = smem_u32(&ctl.empty[r.slot]);
            r.next();
          }
          if (!ok) break;
          tc_fence_after();
          const uint32_t sf = tb + Cfg::kSfCol0 + set * Cfg::kBatch * Cfg::kSfSet;
          if (elect_one()) {
#pragma unroll
            for (int b = 0; b < Cfg::kBatch; ++b) {
              if (k0 + b >= chunks) break;
              const uint32_t sft = sf + b * Cfg::kSfSet, sfw = sft + 4 * Cfg::kWords;
#pragma unroll
              for (int w = 0; w < Cfg::kWords; ++w) {  // (words past a row's last: copied, not used)
                tmem_cp_32x128b_x4_pair(sft + 4 * w, sdesc_sf(st[b] + Cfg::oSt + 512 * w));
                tmem_cp_32x128b_x4_pair(sfw + 8 * w, sdesc_sf(st[b] + Cfg::oSw + 512 * w));
                tmem_cp_32x128b_x4_pair(sfw + 8 * w + 4,
                                        sdesc_sf(st[b] + Cfg::oSw + Cfg::kSf + 512 * w));
              }
            }
#pragma unroll
            for (int b = 0; b < Cfg::kBatch; ++b) {
              const int k = k0 + b;
              if (k >= chunks) break;
              const uint32_t sft = sf + b * Cfg::kSfSet, sfw = sft + 4 * Cfg::kWords;
              const int steps = min(4, (p.K - k * kF4ChunkK + 63) / 64);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                if (kk >= steps) break;
                const int w = kNv ? kk : kk >> 1;
                const uint32_t idesc = idesc_mxf4(256, 256, !kNv, kNv ? 0 : 2 * (kk & 1));
                mma_mxf4_ss<kNv, true>(tb, sdesc_sw128(st[b] + kk * 32),
                                       sdesc_sw128(st[b] + Cfg::oW + kk * 32), idesc, sft + 4 * w,
                                       sfw + 8 * w, (k > 0 || kk > 0) ? 1u : 0u);
              }
              tc_commit_pair(free[b], 3);
              if (k + 1 == chunks) tc_commit_pair(smem_u32(&ctl.acc_full), 3);
            }
          }
          __syncwarp();
          set ^= 1u;
        }
      }
      // arrives once every tcgen05 operation this warp issued has completed
      if (elect_one()) tc_commit_pair(smem_u32(&ctl.drain), 3);
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    const uint32_t acc = tb + (static_cast<uint32_t>(32 * quarter) << 16) + 128 * group;
    const uint32_t acc_empty = mapa_shared(smem_u32(&ctl.acc_empty), 0);
    uint32_t aph = 0;
    grid_dep_wait();  // C, bias and the row scales belong to the previous grid until it ends
    for (int tile = cluster; tile < tiles; tile += clusters) {
      const int m = tile % p.m_tiles * 256 + 128 * static_cast<int>(rank) + 32 * quarter + lane;
      const int n0 = tile / p.m_tiles * 256 + 128 * group;
      const float scale = p.row_scale_t != nullptr && m < p.M
                              ? __fmul_rn(p.row_scale_t[m], p.tensor_scale)
                              : p.tensor_scale;
      if (!__all_sync(0xffffffffu, mbar_wait<true>(smem_u32(&ctl.acc_full), aph, p.err, kErrWaitAccum,
                                                   abort_flag)))
        break;
      aph ^= 1u;
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld_x32(acc + 32 * i, r[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld_wait_x32(r[i]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(acc_empty);
      if (m >= p.M) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + 32 * i;
        if (n >= p.N) break;
        const int64_t at = static_cast<int64_t>(m) * p.N + n;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __fmul_rn(__uint_as_float(r[i][j]), scale);
        if (n + 32 <= p.N) {
          if (p.row_scale_w != nullptr) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __fmul_rn(v[j], p.row_scale_w[n + j]);
          }
          apply_epilogue_row<32>(v, 1.0f, p.epilogue, p.bias, n);
          store_row<32>(p.out, at, v, p.out_dtype, p.vec_out);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (n + j < p.N) {
              float x = p.row_scale_w != nullptr ? __fmul_rn(v[j], p.row_scale_w[n + j]) : v[j];
              store_out(p.out, at + j, apply_epilogue(x, p.epilogue, p.bias, n + j), p.out_dtype);
            }
        }
      }
    }
  }
  // ---- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (lane == 0) mbar_wait(smem_u32(&ctl.drain), 0, p.err, kErrWaitMma, nullptr);
    __syncwarp();
    tc_fence_after();
  }
  // neither CTA frees its tensor memory or exits while the peer may still arrive on its barriers
  cluster_sync_all();
  if (warp == 1) tmem_dealloc_pair(tb, 512);
}

}  // namespace bd
