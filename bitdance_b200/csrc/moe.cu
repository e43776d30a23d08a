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

int last_status() { return cudaPeekAtLastError() == cudaSuccess ? BD_OK : BD_ERR_CUDA; }

// Workspace: counters | row maxima of h | scales of x | fp16 image of x | h | partial sums, each
// 256-byte aligned. Few pairs may split the down product: at least kPartRows rows of partials.
constexpr int kPartRows = 256;
struct MoeWs {
  size_t hmax, x_scale, xs, h, part, total;
  int part_rows;
};
MoeWs moe_ws(int T, int H, int I, int k) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  const size_t pairs = static_cast<size_t>(T) * k;
  MoeWs w;
  w.part_rows = std::max(T * k, kPartRows);
  w.hmax = 256;
  w.x_scale = w.hmax + up(pairs * 4);
  w.xs = w.x_scale + up(static_cast<size_t>(T) * 4);
  w.h = w.xs + up(static_cast<size_t>(T) * H * 2);
  w.part = w.h + up(pairs * I * 4);
  w.total = w.part + static_cast<size_t>(w.part_rows) * H * 4;
  return w;
}

bool bad_shape(int T, int H, int I, int E, int k) {
  return T < 0 || T > kMoeMaxTokens || H <= 0 || I <= 0 || H % 128 || I % 128 || H > (1 << 20) ||
         I > (1 << 20) || E <= 0 || E > kMoeMaxExperts || k <= 0 || k > kMoeMaxTopK || k > E;
}

cudaLaunchConfig_t config(int grid, int smem, cudaStream_t s, cudaLaunchAttribute* attr,
                          int cluster) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kMoeThreads);
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

template <class X, class W, int TB>
int launch_route(const MoeRouteParams& p, cudaStream_t s) {
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config((p.T + TB - 1) / TB * kRouteCluster,
                                        2 * p.E * static_cast<int>(sizeof(double)), s, attr,
                                        kRouteCluster);
  return cudaLaunchKernelEx(&cfg, moe_route_kernel<X, W, TB>, p) == cudaSuccess ? last_status()
                                                                              : BD_ERR_CUDA;
}

template <class X, class W>
int launch_route_t(const MoeRouteParams& p, cudaStream_t s) {
  // tokens per cluster: one while the clusters leave SMs free, more where each pass over the
  // router weights should serve several tokens
  if (p.T <= 16) return launch_route<X, W, 1>(p, s);
  if (p.T <= 32) return launch_route<X, W, 2>(p, s);
  return launch_route<X, W, 4>(p, s);
}

template <int MB>
int launch_experts(const MoeExpertsParams& p, const DeviceInfo* d, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return BD_ERR_CUDA;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    if (cudaFuncSetAttribute(moe_experts_kernel<MB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMoeBBytes) != cudaSuccess)
      return BD_ERR_CUDA;
    configured.fetch_or(bit);
  }
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(2 * d->sm_count, kMoeBBytes, s, attr, 1);
  return cudaLaunchKernelEx(&cfg, moe_experts_kernel<MB>, p) == cudaSuccess ? last_status()
                                                                            : BD_ERR_CUDA;
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
  if (!ws || ws_bytes < moe_ws(T, H, I, k).total) return BD_ERR_WORKSPACE;
  if (!aligned(ws, 256) || !aligned(x, 16) || !aligned(a.w13, 16) || !aligned(a.w2, 16) ||
      !aligned(a.s13, 2) || !aligned(a.s2, 2) || !aligned(a.ts13, 4) || !aligned(a.ts2, 4) ||
      !aligned(ids, 4) || !aligned(weights, 4) || !aligned(y, out_dtype == BD_OUT_F32 ? 4 : 2))
    return BD_ERR_ALIGNMENT;
  return BD_OK;
}

int run_experts(void* y, int out_dtype, const int* ids, const float* weights,
                const MoeExpertArgs& a, int T, int H, int I, int E, int k, uint8_t* ws,
                const DeviceInfo* d, cudaStream_t s) {
  const MoeWs w = moe_ws(T, H, I, k);
  MoeExpertsParams p;
  p.w13 = a.w13;
  p.s13 = a.s13;
  p.ts13 = a.ts13;
  p.w2 = a.w2;
  p.s2 = a.s2;
  p.ts2 = a.ts2;
  p.ids = ids;
  p.weights = weights;
  p.xs = reinterpret_cast<const __half*>(ws + w.xs);
  p.x_scale = reinterpret_cast<const float*>(ws + w.x_scale);
  p.h = reinterpret_cast<float*>(ws + w.h);
  p.hmax = reinterpret_cast<uint32_t*>(ws + w.hmax);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.part_rows = w.part_rows;
  p.vec_out = aligned(y, 16) ? 1 : 0;
  p.y = y;
  p.counters = reinterpret_cast<uint32_t*>(ws);
  p.T = T;
  p.H = H;
  p.I = I;
  p.E = E;
  p.k = k;
  p.out_dtype = out_dtype;
  p.err = d->err;
  // weight rows per task: 256 where the experts that can be touched give the machine two tasks per
  // SM in the gate / up phase, else 128
  const int64_t touched = std::min(E, T * k);
  return touched * (I / 128) >= 2 * d->sm_count ? launch_experts<2>(p, d, s)
                                                : launch_experts<1>(p, d, s);
}

}  // namespace
}  // namespace bd

using namespace bd;

extern "C" {

size_t bd_query_moe_workspace(int T, int H, int I, int E, int top_k) {
  if (bad_shape(T, H, I, E, top_k) || T == 0) return 0;
  return moe_ws(T, H, I, top_k).total;
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
  const MoeWs w = moe_ws(T, H, I, top_k);
  __half* xs = reinterpret_cast<__half*>(ws + w.xs);
  float* x_scale = reinterpret_cast<float*>(ws + w.x_scale);
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws);
  uint32_t* hmax = reinterpret_cast<uint32_t*>(ws + w.hmax);
  cudaStream_t s = as_stream(stream);
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(T, 0, s, attr, 1);
  const cudaError_t e =
      x_dtype == BD_IN_BF16
          ? cudaLaunchKernelEx(&cfg, moe_prepare_kernel<__nv_bfloat16>,
                               static_cast<const __nv_bfloat16*>(x), xs, x_scale, counters, hmax, H,
                               top_k)
          : cudaLaunchKernelEx(&cfg, moe_prepare_kernel<__half>, static_cast<const __half*>(x), xs,
                               x_scale, counters, hmax, H, top_k);
  if (e != cudaSuccess) return BD_ERR_CUDA;
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
  const MoeWs w = moe_ws(T, H, I, top_k);
  MoeRouteParams p;
  p.x = x;
  p.router = router;
  p.bias = selection_bias;
  p.ids = ids;
  p.weights = weights;
  p.xs = reinterpret_cast<__half*>(ws + w.xs);
  p.x_scale = reinterpret_cast<float*>(ws + w.x_scale);
  p.counters = reinterpret_cast<uint32_t*>(ws);
  p.hmax = reinterpret_cast<uint32_t*>(ws + w.hmax);
  p.T = T;
  p.H = H;
  p.E = E;
  p.k = top_k;
  p.sigmoid = scoring == BD_MOE_SIGMOID;
  p.renormalize = renormalize != 0;
  p.routed_scale = routed_scale;
  cudaStream_t s = as_stream(stream);
  if (x_dtype == BD_IN_BF16)
    st = router_dtype == BD_IN_F32 ? launch_route_t<__nv_bfloat16, float>(p, s)
                                   : launch_route_t<__nv_bfloat16, __nv_bfloat16>(p, s);
  else
    st = router_dtype == BD_IN_F32 ? launch_route_t<__half, float>(p, s)
                                   : launch_route_t<__half, __half>(p, s);
  if (st != BD_OK) return st;
  return run_experts(y, out_dtype, ids, weights, a, T, H, I, E, top_k, ws, d, s);
}

}  // extern "C"
