// fp4.cu -- C ABI of the 4-bit operators: quantiser, dequantiser, scale tiles, W4A4 GEMM
// (argument checks, tensor maps and launches of the kernels in fp4.cuh and gemm_fp4.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "fp4.cuh"
#include "gemm_fp4.cuh"
#include "host.cuh"
#include "sm100.cuh"

namespace bd {
namespace {

constexpr int kMaxRows = 1 << 28, kMaxK = 1 << 24;

// Scale tiles (of four scales) along a row of K elements.
int sf_words(int K, int fmt) {
  const int block = fmt == BD_FP4_NVFP4 ? 16 : 32;
  return (K / block + 3) / 4;
}

bool bad_fmt(int fmt) { return fmt != BD_FP4_NVFP4 && fmt != BD_FP4_MXFP4; }

// Raises a kernel's dynamic shared memory limit once per device.
template <class K>
bool allow_smem(K kernel, int bytes, std::atomic<uint64_t>& configured) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (configured.load() & bit) return true;
  if (launch_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)))
    return false;
  configured.fetch_or(bit);
  return true;
}

cudaLaunchConfig_t launch_config(int grid, int threads, int smem, cudaStream_t s,
                                 cudaLaunchAttribute* attr, bool overlap, int cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  if (overlap) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    ++cfg.numAttrs;
  }
  return cfg;
}

template <int kIn, int kFmt>
int launch_quantize(const QuantFp4Params& p, bool overlap, const DeviceInfo* d, cudaStream_t s) {
  cudaLaunchAttribute attr[2];
  const auto launch = [&](auto kernel, int G) {
    const cudaLaunchConfig_t cfg = launch_config(grid_for(p.M, q4_threads(G) / G, d), q4_threads(G), 0,
                                                 s, attr, overlap);
    return cudaLaunchKernelEx(&cfg, kernel, p);
  };
  // A warp per row where rows are short, or many enough for two rounds of a full machine (rows of up to
  // 4096 elements where their maximum comes first: a warp reads what it cannot keep twice); a CTA of
  // four warps where the rows give every SM four; else of eight. Measured, bf16: 8192 x 4096 NVFP4
  // 28 / 36 / 43 us, 8192 x 14336 MXFP4 63 / 70 / 63, 2048 x 8192 NVFP4 17 / 14 / 17, 600 x 4096 NVFP4
  // 7.4 / 4.0 / 4.8; fp32: 4099 x 14336 NVFP4 86 / 68 / 69, MXFP4 50 / 47 / 50.
  const bool warp_rows =
      p.K <= 1024 || (p.M >= 32 * d->sm_count && (kFmt == kMxfp4 || p.K <= 4096));
  const cudaError_t e = warp_rows                ? launch(quantize_fp4_kernel<kIn, kFmt, 32>, 32)
                        : p.M >= 4 * d->sm_count ? launch(quantize_fp4_kernel<kIn, kFmt, 128>, 128)
                                                 : launch(quantize_fp4_kernel<kIn, kFmt, 256>, 256);
  return launch_status(e);
}

template <int kFmt>
int launch_quantize_in(int in, const QuantFp4Params& p, bool overlap, const DeviceInfo* d,
                       cudaStream_t s) {
  if (in == BD_IN_F32) return launch_quantize<kInF32, kFmt>(p, overlap, d, s);
  if (in == BD_IN_BF16) return launch_quantize<kInBf16, kFmt>(p, overlap, d, s);
  return launch_quantize<kInF16, kFmt>(p, overlap, d, s);
}

template <int kFmt, int kOut>
int launch_dequantize(const uint8_t* codes, const uint8_t* tiled, const float* rs, float ts,
                      void* out, int M, int K, bool overlap, const DeviceInfo* d,
                      cudaStream_t s) {
  const bool warp_rows = K <= 1024;  // a warp per row, else a CTA
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      launch_config(grid_for(M, warp_rows ? 8 : 1, d), 256, 0, s, attr, overlap);
  uint8_t* o = static_cast<uint8_t*>(out);
  const int words = sf_words(K, kFmt);
  const cudaError_t e =
      warp_rows ? cudaLaunchKernelEx(&cfg, dequantize_fp4_kernel<kFmt, kOut, 32>, codes, tiled, rs,
                                     ts, o, M, K, words)
                : cudaLaunchKernelEx(&cfg, dequantize_fp4_kernel<kFmt, kOut, 256>, codes, tiled, rs,
                                     ts, o, M, K, words);
  return launch_status(e);
}

template <int kFmt>
int launch_dequantize_out(int out_dtype, const uint8_t* codes, const uint8_t* tiled,
                          const float* rs, float ts, void* out, int M, int K, bool overlap,
                          const DeviceInfo* d, cudaStream_t s) {
  if (out_dtype == BD_OUT_BF16)
    return launch_dequantize<kFmt, 0>(codes, tiled, rs, ts, out, M, K, overlap, d, s);
  if (out_dtype == BD_OUT_F16)
    return launch_dequantize<kFmt, 1>(codes, tiled, rs, ts, out, M, K, overlap, d, s);
  return launch_dequantize<kFmt, 2>(codes, tiled, rs, ts, out, M, K, overlap, d, s);
}

bool codes_map(CUtensorMap* m, const uint8_t* codes, int rows, int K, int box_rows) {
  return make_map_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<uint8_t*>(codes), K / 2, rows,
                     K / 2, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Scale tiles as rows of 512 bytes (one word of 128 rows), boxes of box_words of them.
bool scales_map(CUtensorMap* m, const uint8_t* sf, int rows, int words, int box_words) {
  return make_map_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, const_cast<uint8_t*>(sf), 128,
                     (static_cast<uint64_t>(rows) + 127) / 128 * words, 512, 128, box_words,
                     CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int BN, int kFmt>
int launch_gemm(GemmFp4Params p, const uint8_t* a, const uint8_t* b, bool overlap,
                const DeviceInfo* d, cudaStream_t s) {
  using Cfg = GemmFp4Cfg<BN, kFmt>;
  static std::atomic<uint64_t> configured{0};
  if (!allow_smem(w4a4_gemm_kernel<BN, kFmt>, Cfg::kSmemBytes, configured)) return BD_ERR_CUDA;
  p.n_tiles = (p.N + 127) / 128;
  p.m_tiles = (p.M + BN - 1) / BN;
  const int64_t tiles = static_cast<int64_t>(p.n_tiles) * p.m_tiles;
  // K slices per tile (a cluster): doubled while the CTAs still fit the machine at once and each keeps a
  // chunk of its own
  const int chunks = (p.K + kF4ChunkK - 1) / kF4ChunkK;
  int split = 1;
  while (split < 8 && tiles * split * 2 <= static_cast<int64_t>(d->sm_count) * Cfg::kCtasPerSm &&
         chunks >= split * 2)
    split *= 2;
  if (tiles * split > 0x7FFFFFFF) return BD_ERR_SHAPE;
  CUtensorMap mw, mt;
  if (!codes_map(&mw, b, p.N, p.K, 128) || !codes_map(&mt, a, p.M, p.K, BN)) return BD_ERR_CUDA;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = launch_config(static_cast<int>(tiles * split), 128,
                                               Cfg::kSmemBytes, s, attr, overlap, split);
  return launch_status(cudaLaunchKernelEx(&cfg, w4a4_gemm_kernel<BN, kFmt>, mw, mt, p, split));
}

template <int kFmt>
int launch_pair(GemmFp4Params p, const uint8_t* a, const uint8_t* b, bool overlap,
                const DeviceInfo* d, cudaStream_t s) {
  using Cfg = PairFp4Cfg<kFmt>;
  static std::atomic<uint64_t> configured{0};
  if (!allow_smem(w4a4_pair_kernel<kFmt>, Cfg::kSmem, configured)) return BD_ERR_CUDA;
  p.n_tiles = (p.N + 255) / 256;
  p.m_tiles = (p.M + 255) / 256;
  const int64_t tiles = static_cast<int64_t>(p.n_tiles) * p.m_tiles;
  if (tiles > 0x7FFFFFFF) return BD_ERR_SHAPE;
  CUtensorMap mw, mt, sw, st;
  if (!codes_map(&mw, b, p.N, p.K, 128) || !codes_map(&mt, a, p.M, p.K, 128) ||
      !scales_map(&sw, p.sf_w, p.N, p.words, Cfg::kWords) ||
      !scales_map(&st, p.sf_t, p.M, p.words, Cfg::kWords))
    return BD_ERR_CUDA;
  const int grid = 2 * static_cast<int>(std::min<int64_t>(tiles, d->sm_count / 2));
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      launch_config(grid, kPairThreads, Cfg::kSmem, s, attr, overlap, 2);
  return launch_status(cudaLaunchKernelEx(&cfg, w4a4_pair_kernel<kFmt>, mw, mt, sw, st, p));
}

template <int kFmt>
int launch_gemm_any(const GemmFp4Params& p, const uint8_t* a, const uint8_t* b, bool overlap,
                    const DeviceInfo* d, cudaStream_t s) {
  // 256 x 256 tiles where they occupy at least half of the SM pairs: 256 x 14336 x 4096 (56 tiles)
  // 18.9 us for 26.5, 1024 x 4096 x 4096 (64) 16.3 for 25.3; 512 x 4096 x 4096 (32) would take 14.6 for
  // 12.9, 256 x 2048 x 14336 (8) 30 for 17
  const int64_t pair_tiles =
      static_cast<int64_t>((p.N + 255) / 256) * ((p.M + 255) / 256);
  if (p.M > 128 && 4 * pair_tiles >= d->sm_count) return launch_pair<kFmt>(p, a, b, overlap, d, s);
  // else the smallest token tile that holds the batch (several tiles are of 128: a tile's scales are
  // whole 128-row blocks)
  if (p.M <= 16) return launch_gemm<16, kFmt>(p, a, b, overlap, d, s);
  if (p.M <= 32) return launch_gemm<32, kFmt>(p, a, b, overlap, d, s);
  if (p.M <= 64) return launch_gemm<64, kFmt>(p, a, b, overlap, d, s);
  return launch_gemm<128, kFmt>(p, a, b, overlap, d, s);
}

int check_gemm(const void* c, const void* bias, int M, int N, int K, int fmt, int out_dtype,
               int epilogue, const void* b, const void* b_scales, const void* b_row_scale) {
  if (bad_fmt(fmt) || out_dtype < BD_OUT_BF16 || out_dtype > BD_OUT_F32) return BD_ERR_INVALID_ARG;
  if (epilogue < BD_EPI_NONE || epilogue > BD_EPI_BIAS_GELU) return BD_ERR_INVALID_ARG;
  if (M < 0 || N <= 0 || K <= 0 || K % 32 || M > kMaxRows || N > kMaxK || K > kMaxK)
    return BD_ERR_SHAPE;
  if (M == 0) return BD_OK;
  if (!c || !b || !b_scales || (epilogue != BD_EPI_NONE && !bias)) return BD_ERR_INVALID_ARG;
  if (!aligned(b, 16) || !aligned(b_scales, 16) || (b_row_scale && !aligned(b_row_scale, 4)) ||
      (bias && !aligned(bias, 2)) || !aligned(c, out_dtype == BD_OUT_F32 ? 4 : 2))
    return BD_ERR_ALIGNMENT;
  return BD_OK;
}

// bd_quantize_fp4; release: as in QuantFp4Params.
int quantize(const void* x, int x_dtype, int fmt, uint8_t* codes, uint8_t* scales,
             uint8_t* scales_tiled, float* row_scale, int M, int K, bool overlap,
             bool release, bd_stream_t stream) {
  if (bad_fmt(fmt) || x_dtype < BD_IN_F32 || x_dtype > BD_IN_F16) return BD_ERR_INVALID_ARG;
  if (M < 0 || K <= 0 || K % 32 || M > kMaxRows || K > kMaxK) return BD_ERR_SHAPE;
  if (M == 0) return BD_OK;
  if (!x || !codes || (!scales && !scales_tiled)) return BD_ERR_INVALID_ARG;
  if (fmt == BD_FP4_NVFP4 && !row_scale) return BD_ERR_INVALID_ARG;
  if (!aligned(x, 16) || !aligned(codes, 16) || (scales_tiled && !aligned(scales_tiled, 16)) ||
      (row_scale && !aligned(row_scale, 4)))
    return BD_ERR_ALIGNMENT;
  DeviceInfo* d = nullptr;
  const int st = device_info(&d);
  if (st != BD_OK) return st;
  const QuantFp4Params p{x, codes, scales, scales_tiled, row_scale, M, K, sf_words(K, fmt),
                         release ? 1 : 0, d->err};
  return fmt == BD_FP4_NVFP4
             ? launch_quantize_in<kNvfp4>(x_dtype, p, overlap, d, as_stream(stream))
             : launch_quantize_in<kMxfp4>(x_dtype, p, overlap, d, as_stream(stream));
}

// Workspace of bd_w4a4_linear: codes | scale tiles | row scales, each 256-byte aligned.
struct LinearWs {
  size_t codes, scales, total;
};
LinearWs linear_ws(int M, int K, int fmt) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  LinearWs w;
  w.codes = up(static_cast<size_t>(M) * (K / 2));
  w.scales = w.codes + up(bd_query_fp4_scales(M, K, fmt));
  w.total = w.scales + up(static_cast<size_t>(M) * sizeof(float));
  return w;
}

}  // namespace
}  // namespace bd

using namespace bd;

extern "C" {

size_t bd_query_fp4_scales(int rows, int K, int fmt) {
  if (bad_fmt(fmt) || rows <= 0 || K <= 0 || K % 32) return 0;
  return (static_cast<size_t>(rows) + 127) / 128 * static_cast<size_t>(sf_words(K, fmt)) * 512;
}

int bd_quantize_fp4(const void* x, int x_dtype, int fmt, uint8_t* codes, uint8_t* scales,
                    uint8_t* scales_tiled, float* row_scale, int M, int K, unsigned flags,
                    bd_stream_t stream) {
  if (flags & ~static_cast<unsigned>(BD_GEMM_OVERLAP_PREV)) return BD_ERR_INVALID_ARG;
  return quantize(x, x_dtype, fmt, codes, scales, scales_tiled, row_scale, M, K,
                  (flags & BD_GEMM_OVERLAP_PREV) != 0, false, stream);
}

int bd_tile_scales_fp4(const uint8_t* scales, uint8_t* scales_tiled, int rows, int K, int fmt,
                       bd_stream_t stream) {
  if (bad_fmt(fmt)) return BD_ERR_INVALID_ARG;
  if (rows < 0 || K <= 0 || K % 32 || rows > kMaxRows || K > kMaxK) return BD_ERR_SHAPE;
  if (rows == 0) return BD_OK;
  if (!scales || !scales_tiled) return BD_ERR_INVALID_ARG;
  if (!aligned(scales_tiled, 16)) return BD_ERR_ALIGNMENT;
  DeviceInfo* d = nullptr;
  const int st = device_info(&d);
  if (st != BD_OK) return st;
  const int words = sf_words(K, fmt);
  const int64_t work = static_cast<int64_t>(rows) * words;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      launch_config(grid_for(work, 256, d), 256, 0, as_stream(stream), attr, false);
  return launch_status(cudaLaunchKernelEx(&cfg, tile_scales_kernel, scales, scales_tiled, rows,
                                          K / (fmt == BD_FP4_NVFP4 ? 16 : 32), words));
}

int bd_dequantize_fp4(const uint8_t* codes, const uint8_t* scales_tiled, const float* row_scale,
                      float tensor_scale, void* out, int out_dtype, int fmt, int M, int K,
                      unsigned flags, bd_stream_t stream) {
  if (flags & ~static_cast<unsigned>(BD_GEMM_OVERLAP_PREV)) return BD_ERR_INVALID_ARG;
  if (bad_fmt(fmt) || out_dtype < BD_OUT_BF16 || out_dtype > BD_OUT_F32) return BD_ERR_INVALID_ARG;
  if (M < 0 || K <= 0 || K % 32 || M > kMaxRows || K > kMaxK) return BD_ERR_SHAPE;
  if (M == 0) return BD_OK;
  if (!codes || !scales_tiled || !out) return BD_ERR_INVALID_ARG;
  if (!aligned(codes, 8) || !aligned(out, 16) || (row_scale && !aligned(row_scale, 4)))
    return BD_ERR_ALIGNMENT;
  DeviceInfo* d = nullptr;
  const int st = device_info(&d);
  if (st != BD_OK) return st;
  const bool overlap = (flags & BD_GEMM_OVERLAP_PREV) != 0;
  return fmt == BD_FP4_NVFP4
             ? launch_dequantize_out<kNvfp4>(out_dtype, codes, scales_tiled, row_scale, tensor_scale,
                                         out, M, K, overlap, d, as_stream(stream))
             : launch_dequantize_out<kMxfp4>(out_dtype, codes, scales_tiled, row_scale, tensor_scale,
                                         out, M, K, overlap, d, as_stream(stream));
}

int bd_w4a4_gemm(void* c, const uint8_t* a, const uint8_t* a_scales, const float* a_row_scale,
                 const uint8_t* b, const uint8_t* b_scales, const float* b_row_scale,
                 float tensor_scale, const void* bias, int M, int N, int K, int fmt,
                 int out_dtype, int epilogue, unsigned flags, bd_stream_t stream) {
  if (flags & ~static_cast<unsigned>(BD_GEMM_OVERLAP_PREV | BD_GEMM_WEIGHTS_STATIC))
    return BD_ERR_INVALID_ARG;
  int st = check_gemm(c, bias, M, N, K, fmt, out_dtype, epilogue, b, b_scales, b_row_scale);
  if (st != BD_OK || M == 0) return st;
  if (!a || !a_scales) return BD_ERR_INVALID_ARG;
  if (!aligned(a, 16) || !aligned(a_scales, 16) || (a_row_scale && !aligned(a_row_scale, 4)))
    return BD_ERR_ALIGNMENT;
  DeviceInfo* d = nullptr;
  st = device_info(&d);
  if (st != BD_OK) return st;
  GemmFp4Params p = {};
  p.out = c;
  p.sf_t = a_scales;
  p.sf_w = b_scales;
  p.row_scale_t = a_row_scale;
  p.row_scale_w = b_row_scale;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.tensor_scale = tensor_scale;
  p.M = M;
  p.N = N;
  p.K = K;
  p.words = sf_words(K, fmt);
  p.out_dtype = out_dtype;
  p.epilogue = epilogue;
  p.vec_out = aligned(c, 16) && static_cast<int64_t>(N) * (out_dtype == BD_OUT_F32 ? 4 : 2) % 16 == 0;
  p.weights_early = (flags & BD_GEMM_WEIGHTS_STATIC) ? 1 : 0;
  p.err = d->err;
  const bool overlap = (flags & BD_GEMM_OVERLAP_PREV) != 0;
  return fmt == BD_FP4_NVFP4 ? launch_gemm_any<kNvfp4>(p, a, b, overlap, d, as_stream(stream))
                             : launch_gemm_any<kMxfp4>(p, a, b, overlap, d, as_stream(stream));
}

int bd_selftest_cluster_wait(int64_t limit_cycles, int ctas, int failing, uint32_t* stored,
                             bd_stream_t stream) {
  if (limit_cycles < 1000 || static_cast<unsigned long long>(limit_cycles) > kWaitLimitCycles)
    return BD_ERR_INVALID_ARG;
  if ((ctas != 2 && ctas != 4 && ctas != 8) || failing < -1 || failing >= ctas || !stored)
    return BD_ERR_INVALID_ARG;
  if (!aligned(stored, 4)) return BD_ERR_ALIGNMENT;
  DeviceInfo* d = nullptr;
  const int st = device_info(&d);
  if (st != BD_OK) return st;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = launch_config(ctas, 128, 0, as_stream(stream), attr, false, ctas);
  return launch_status(cudaLaunchKernelEx(&cfg, cluster_wait_selftest_kernel, stored, ctas, failing,
                                          static_cast<unsigned long long>(limit_cycles), d->err));
}

size_t bd_query_w4a4_linear_workspace(int M, int K, int fmt) {
  if (bad_fmt(fmt) || M <= 0 || K <= 0 || K % 32) return 0;
  return linear_ws(M, K, fmt).total;
}

int bd_w4a4_linear(void* c, const void* x, int x_dtype, const uint8_t* b, const uint8_t* b_scales,
                   const float* b_row_scale, float tensor_scale, const void* bias, int M, int N,
                   int K, int fmt, int out_dtype, int epilogue, void* workspace,
                   size_t workspace_bytes, bd_stream_t stream) {
  if (x_dtype < BD_IN_F32 || x_dtype > BD_IN_F16) return BD_ERR_INVALID_ARG;
  int st = check_gemm(c, bias, M, N, K, fmt, out_dtype, epilogue, b, b_scales, b_row_scale);
  if (st != BD_OK || M == 0) return st;
  if (!x) return BD_ERR_INVALID_ARG;
  const LinearWs w = linear_ws(M, K, fmt);
  if (!workspace || workspace_bytes < w.total) return BD_ERR_WORKSPACE;
  if (!aligned(workspace, 256) || !aligned(x, 16)) return BD_ERR_ALIGNMENT;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* row_scale = fmt == BD_FP4_NVFP4 ? reinterpret_cast<float*>(ws + w.scales) : nullptr;
  st = quantize(x, x_dtype, fmt, ws, nullptr, ws + w.codes, row_scale, M, K, true, true, stream);
  if (st != BD_OK) return st;
  return bd_w4a4_gemm(c, ws, ws + w.codes, row_scale, b, b_scales, b_row_scale, tensor_scale, bias,
                      M, N, K, fmt, out_dtype, epilogue,
                      BD_GEMM_OVERLAP_PREV | BD_GEMM_WEIGHTS_STATIC, stream);
}

}  // extern "C"
