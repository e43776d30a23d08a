// epilogue.cuh -- scale, bias, activation and output conversion shared by the GEMM kernels.
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace bd {

// SiLU and tanh-GELU with every multiply and add rounded on its own (no contraction into FMAs,
// which the compiler may do differently in different drain loops): every store path of the
// GEMM gives the same bits.
__device__ __forceinline__ float silu_rn(float v) {
  return __fdiv_rn(v, __fadd_rn(1.0f, expf(-v)));
}
__device__ __forceinline__ float gelu_tanh_rn(float v) {
  const float v3 = __fmul_rn(__fmul_rn(v, v), v);
  const float y = __fmul_rn(0.7978845608028654f, __fadd_rn(v, __fmul_rn(0.044715f, v3)));
  return __fmul_rn(__fmul_rn(0.5f, v), __fadd_rn(1.0f, tanhf(y)));
}

__device__ __forceinline__ float apply_epilogue(float v, int epi, const __nv_bfloat16* bias,
                                                int n) {
  if (epi != 0) v = __fadd_rn(v, __bfloat162float(bias[n]));
  if (epi == 2) v = fmaxf(v, 0.0f);
  else if (epi == 3) v = silu_rn(v);
  else if (epi == 4) v = gelu_tanh_rn(v);
  return v;
}

// The same for NV consecutive outputs n .. n + NV - 1, scaled first: the epilogue kind is
// tested once per row piece, not per element (a per-element test in an unrolled drain loop
// cost more than the conversion itself), with the same operations in the same order.
template <int NV>
__device__ __forceinline__ void apply_epilogue_row(float (&v)[NV], float scale, int epi,
                                                   const __nv_bfloat16* bias, int n) {
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = __fmul_rn(v[j], scale);
  if (epi == 0) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = __fadd_rn(v[j], __bfloat162float(bias[n + j]));
  if (epi == 2) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = fmaxf(v[j], 0.0f);
  } else if (epi == 3) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = silu_rn(v[j]);
  } else if (epi == 4) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = gelu_tanh_rn(v[j]);
  }
}

__device__ __forceinline__ void store_out(void* out, int64_t idx, float v, int dtype) {
  if (dtype == 0) reinterpret_cast<__nv_bfloat16*>(out)[idx] = __float2bfloat16_rn(v);
  else if (dtype == 1) reinterpret_cast<__half*>(out)[idx] = __float2half_rn(v);
  else reinterpret_cast<float*>(out)[idx] = v;
}

// NV consecutive outputs (element index idx, a multiple of NV) in the output dtype; vector
// stores (16 bytes, 8 for four 16-bit values) when C is 16-byte aligned.
template <int NV>
__device__ __forceinline__ void store_row(void* out, int64_t idx, const float (&v)[NV], int dtype,
                                          int vec) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < NV; ++j) store_out(out, idx + j, v[j], dtype);
    return;
  }
  if (dtype == 2) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + idx);
#pragma unroll
    for (int j = 0; j < NV / 4; ++j)
      o[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    return;
  }
  uint32_t w[NV / 2];
#pragma unroll
  for (int j = 0; j < NV / 2; ++j) {
    if (dtype == 0) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  if constexpr (NV % 8 == 0) {
    uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + idx);
#pragma unroll
    for (int j = 0; j < NV / 8; ++j)
      o[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  } else {
    static_assert(NV == 4, "4, 8, 16 or 32 outputs");
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + idx) = make_uint2(w[0], w[1]);
  }
}

}  // namespace bd
