// moe.cu -- C ABI of the mixture-of-experts layer (argument checks and launches of the kernels in
// moe.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "host.cuh"
#include "moe.cuh"

namespace bd {
namespace {

// Workspace: counters | row maxima of h | row factors of x | digits of x | h | digits of h | partial
// sums, each 256-byte aligned. Few pairs may split the down product: at least kPartRows rows of
// partials.
constexpr int kPartRows = 256;
struct MoeWs {
  size_t hmax, x_scale, xs, h, hs, part, total;
  int part_rows;
};
MoeWs moe_ws(int T, int H, int I, int E, int k) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  const size_t pairs = static_cast<size_t>(T) * k;
  MoeWs w;
  w.part_rows = std::max(T * k, kPartRows);
  w.hmax = up(static_cast<size_t>(moe_counters(E)) * 4);
  w.x_scale = w.hmax + up(pairs * 4);
  w.xs = w.x_scale + up(static_cast<size_t>(T) * 4);
  w.h = w.xs + up(T * moe_image_row(H));
  w.hs = w.h + up(pairs * I * 4);
  w.part = w.hs + up(pairs * moe_image_row(I));
  w.total = w.part + static_cast<size_t>(w.part_rows) * H * 4;
  return w;
}

bool bad_shape(int T, int H, int I, int E, int k) {
  return T < 0 || T > kMoeMaxTokens || H <= 0 || I <= 0 || H % 128 || I % 128 || H > (1 << 20) ||
         I > (1 << 20) || E <= 0 || E > kMoeMaxExperts || k <= 0 || k > kMoeMaxTopK || k > E ||
         static_cast<int64_t>(E) * std::max(H, 2 * I) > 0x7FFFFFFF;
}

cudaLaunchConfig_t config(int grid, int threads, int smem, cudaStream_t s, cudaLaunchAttribute* attr,
                          int cluster) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    cfg.numAttrs = 2;
  }
  return cfg;
}

template <class X, class W, int parts>
int launch_route_parts(const MoeRouteParams& p, cudaStream_t s) {
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      config(p.T * kRouteCluster, kMoeThreads, (parts + 1) * p.E * static_cast<int>(sizeof(double)), s,
             attr, kRouteCluster);
  return launch_status(cudaLaunchKernelEx(&cfg, moe_route_kernel<X, W, parts>, p));
}

// Eight parts of K per expert where one warp per expert leaves most of a CTA's warps idle (rows shorter
// than one round of 8 x 32 lanes x 8 elements have nothing to split). The layer with 8 experts, H 4096,
// 8 / 32 / 64 tokens: 47 / 51 / 63 us for 50 / 53 / 69 in one part; with 32 of H 2048 equal; with 64 of
// H 4096, 8 / 64 tokens: 80 / 125 for 76 / 119.
template <class X, class W>
int launch_route(const MoeRouteParams& p, cudaStream_t s) {
  return p.E <= 4 * kRouteCluster && p.H >= 2048 ? launch_route_parts<X, W, 8>(p, s)
                                                 : launch_route_parts<X, W, 1>(p, s);
}

struct MoeExpertArgs {
  const uint8_t* w13;
  const uint8_t* s13;
  const float* ts13;
  const uint8_t* w2;
  const uint8_t* s2;
  const float* ts2;
};

int check_experts(const void* y, const void* x, int x_dtype, int out_dtype, const int* ids,
                  const float* weights, const MoeExpertArgs& a, int T, int H, int I, int E, int k,
                  const void* ws, size_t ws_bytes) {
  if (x_dtype != BD_IN_BF16 && x_dtype != BD_IN_F16) return BD_ERR_INVALID_ARG;
  if (out_dtype < BD_OUT_BF16 || out_dtype > BD_OUT_F32) return BD_ERR_INVALID_ARG;
  if (bad_shape(T, H, I, E, k)) return BD_ERR_SHAPE;
  if (T == 0) return BD_OK;
  if (!y || !x || !ids || !weights || !a.w13 || !a.s13 || !a.ts13 || !a.w2 || !a.s2 || !a.ts2)
    return BD_ERR_INVALID_ARG;
  if (!ws || ws_bytes < moe_ws(T, H, I, E, k).total) return BD_ERR_WORKSPACE;
  if (!aligned(ws, 256) || !aligned(x, 16) || !aligned(a.w13, 16) || !aligned(a.w2, 16) ||
      !aligned(a.s13, 8) || !aligned(a.s2, 8) || !aligned(a.ts13, 4) || !aligned(a.ts2, 4) ||
      !aligned(ids, 4) || !aligned(weights, 4) || !aligned(y, out_dtype == BD_OUT_F32 ? 4 : 2))
    return BD_ERR_ALIGNMENT;
  return BD_OK;
}

bool codes_map(CUtensorMap* m, const uint8_t* codes, int64_t rows, int K) {
  return make_map_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<uint8_t*>(codes), K / 2, rows,
                     K / 2, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int TOK>
int launch_experts(const CUtensorMap& m13, const CUtensorMap& m2, const MoeExpertsParams& p,
                   const DeviceInfo* d, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return BD_ERR_CUDA;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    const int st = launch_status(cudaFuncSetAttribute(
        moe_experts_kernel<TOK>, cudaFuncAttributeMaxDynamicSharedMemorySize, MoeCfg<TOK>::kSmem));
    if (st != BD_OK) return st;
    configured.fetch_or(bit);
  }
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      config(d->sm_count, kMoeExpertThreads, MoeCfg<TOK>::kSmem, s, attr, 1);
  return launch_status(cudaLaunchKernelEx(&cfg, moe_experts_kernel<TOK>, m13, m2, p));
}

int run_experts(void* y, int out_dtype, const int* ids, const float* weights,
                const MoeExpertArgs& a, int T, int H, int I, int E, int k, uint8_t* ws,
                const DeviceInfo* d, cudaStream_t s) {
  const MoeWs w = moe_ws(T, H, I, E, k);
  MoeExpertsParams p;
  p.s13 = a.s13;
  p.s2 = a.s2;
  p.ts13 = a.ts13;
  p.ts2 = a.ts2;
  p.ids = ids;
  p.weights = weights;
  p.xs = ws + w.xs;
  p.x_scale = reinterpret_cast<const float*>(ws + w.x_scale);
  p.h = reinterpret_cast<float*>(ws + w.h);
  p.hmax = reinterpret_cast<uint32_t*>(ws + w.hmax);
  p.hs = ws + w.hs;
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.y = y;
  p.counters = reinterpret_cast<uint32_t*>(ws);
  p.T = T;
  p.H = H;
  p.I = I;
  p.E = E;
  p.k = k;
  p.part_rows = w.part_rows;
  p.out_dtype = out_dtype;
  p.vec_out = aligned(y, 16) ? 1 : 0;
  p.err = d->err;
  CUtensorMap m13, m2;
  if (!codes_map(&m13, a.w13, static_cast<int64_t>(E) * 2 * I, H) ||
      !codes_map(&m2, a.w2, static_cast<int64_t>(E) * H, I))
    return BD_ERR_CUDA;
  // passes of 16 tokens (half the MMAs) where an expert is expected to have at most about ten, of 24
  // else; an expert with more takes several passes either way. 32 experts of 2048 x 1024 with 8 / 10 /
  // 12 / 16 tokens each: 50 / 55 / 60 / 68 us in passes of 16, 56 / 55 / 57 / 62 us of 24
  return T <= 16 || T * k <= 10 * E ? launch_experts<16>(m13, m2, p, d, s)
                                    : launch_experts<24>(m13, m2, p, d, s);
}

}  // namespace
}  // namespace bd

using namespace bd;

extern "C" {

size_t bd_query_moe_workspace(int T, int H, int I, int E, int top_k) {
  if (bad_shape(T, H, I, E, top_k) || T == 0) return 0;
  return moe_ws(T, H, I, E, top_k).total;
}

int bd_moe_experts(void* y, const void* x, int x_dtype, const int* ids, const float* weights,
                   const uint8_t* gate_up, const uint8_t* gate_up_scales,
                   const float* gate_up_tensor_scale, const uint8_t* down,
                   const uint8_t* down_scales, const float* down_tensor_scale, int T, int H,
                   int I, int E, int top_k, int out_dtype, void* workspace,
                   size_t workspace_bytes, bd_stream_t stream) {
  const MoeExpertArgs a{gate_up, gate_up_scales, gate_up_tensor_scale, down, down_scales,
                        down_tensor_scale};
  int st = check_experts(y, x, x_dtype, out_dtype, ids, weights, a, T, H, I, E, top_k, workspace,
                         workspace_bytes);
  if (st != BD_OK || T == 0) return st;
  DeviceInfo* d = nullptr;
  st = device_info(&d);
  if (st != BD_OK) return st;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const MoeWs w = moe_ws(T, H, I, E, top_k);
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws);
  uint32_t* hmax = reinterpret_cast<uint32_t*>(ws + w.hmax);
  float* x_scale = reinterpret_cast<float*>(ws + w.x_scale);
  cudaStream_t s = as_stream(stream);
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(T, kMoeThreads, 0, s, attr, 1);
  const cudaError_t e =
      x_dtype == BD_IN_BF16
          ? cudaLaunchKernelEx(&cfg, moe_prepare_kernel<__nv_bfloat16>,
                               static_cast<const __nv_bfloat16*>(x), ws + w.xs, x_scale, hmax, counters,
                               H, E, top_k)
          : cudaLaunchKernelEx(&cfg, moe_prepare_kernel<__half>, static_cast<const __half*>(x),
                               ws + w.xs, x_scale, hmax, counters, H, E, top_k);
  if (e != cudaSuccess) return launch_status(e);
  return run_experts(y, out_dtype, ids, weights, a, T, H, I, E, top_k, ws, d, s);
}

int bd_moe_layer(void* y, int* ids, float* weights, const void* x, int x_dtype,
                 const void* router, int router_dtype, const float* selection_bias, int scoring,
                 int renormalize, float routed_scale, const uint8_t* gate_up,
                 const uint8_t* gate_up_scales, const float* gate_up_tensor_scale,
                 const uint8_t* down, const uint8_t* down_scales, const float* down_tensor_scale,
                 int T, int H, int I, int E, int top_k, int out_dtype, void* workspace,
                 size_t workspace_bytes, bd_stream_t stream) {
  const MoeExpertArgs a{gate_up, gate_up_scales, gate_up_tensor_scale, down, down_scales,
                        down_tensor_scale};
  if (scoring != BD_MOE_SOFTMAX && scoring != BD_MOE_SIGMOID) return BD_ERR_INVALID_ARG;
  if (router_dtype != BD_IN_F32 && router_dtype != x_dtype) return BD_ERR_INVALID_ARG;
  int st = check_experts(y, x, x_dtype, out_dtype, ids, weights, a, T, H, I, E, top_k, workspace,
                         workspace_bytes);
  if (st != BD_OK || T == 0) return st;
  if (!router) return BD_ERR_INVALID_ARG;
  if (!aligned(router, 16) || (selection_bias && !aligned(selection_bias, 4)))
    return BD_ERR_ALIGNMENT;
  DeviceInfo* d = nullptr;
  st = device_info(&d);
  if (st != BD_OK) return st;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const MoeWs w = moe_ws(T, H, I, E, top_k);
  MoeRouteParams p;
  p.x = x;
  p.router = router;
  p.bias = selection_bias;
  p.ids = ids;
  p.weights = weights;
  p.xs = ws + w.xs;
  p.x_scale = reinterpret_cast<float*>(ws + w.x_scale);
  p.hmax = reinterpret_cast<uint32_t*>(ws + w.hmax);
  p.counters = reinterpret_cast<uint32_t*>(ws);
  p.T = T;
  p.H = H;
  p.E = E;
  p.k = top_k;
  p.sigmoid = scoring == BD_MOE_SIGMOID;
  p.renormalize = renormalize != 0;
  p.routed_scale = routed_scale;
  cudaStream_t s = as_stream(stream);
  if (x_dtype == BD_IN_BF16)
    st = router_dtype == BD_IN_F32 ? launch_route<__nv_bfloat16, float>(p, s)
                                   : launch_route<__nv_bfloat16, __nv_bfloat16>(p, s);
  else
    st = router_dtype == BD_IN_F32 ? launch_route<__half, float>(p, s)
                                   : launch_route<__half, __half>(p, s);
  if (st != BD_OK) return st;
  return run_experts(y, out_dtype, ids, weights, a, T, H, I, E, top_k, ws, d, s);
}

}  // extern "C"
