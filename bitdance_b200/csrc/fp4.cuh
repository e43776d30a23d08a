// fp4.cuh -- microscaled 4-bit floating point on the GPU: quantiser, dequantiser and scale
// tiling of the operands of the W4A4 GEMM (gemm_fp4.cuh).
//
// Formats (codes E2M1, two per byte along K, element 2j in the low nibble):
//   NVFP4: one E4M3 scale per 16 elements and one fp32 scale per row;
//   MXFP4: one E8M0 scale per 32 elements.
//
// Rule of the NVFP4 quantiser, every step in float32 round-to-nearest:
//   s_m = max(amax(|x_m|) / 2688, 2^-120), 1 for a zero row;  i_m = 1 / s_m
//   per 16-block: top = amax(|x|) * i_m;  B = the smallest E4M3 normal with 6 B >= top (448 at
//   most, 1 for a zero block);  code = nearest E2M1 of x * (i_m / B), a tie to the lower
//   magnitude, the sign only on non-zero codes.
// The row scale makes a token's codes independent of the other tokens of the batch, and one
// row's maximum is a reduction inside one CTA. Two reciprocals, one per row and one per block,
// replace the division per element of the weight quantiser (quantize_b.cuh).
// Rule of the MXFP4 quantiser (the MXFP6 quantiser's with E2M1 in place of E2M3): e the smallest
// integer in [-40, 40] with 6 * 2^e >= amax of the 32-block (0 for a zero block), code = nearest
// E2M1 of x * 2^-e, a tie to the lower magnitude. x * 2^-e is exact (values that leave the normal
// range are far below the first midpoint).
//
// Element code: y = x * r rounded to float32 goes through the hardware's conversion to E2M1, which
// rounds to nearest, a tie to the even code. A tie always has its low 21 mantissa bits zero, and so
// does every E2M1 value; a y with those bits zero is first multiplied by 1 - 2^-24, which takes it to
// the float below: a tie then rounds down, an E2M1 value back to itself. (Integer rounding on float
// bits instead took 11 instructions an element for 6, and the quantiser was bound by them.)
//
// Scale tiles (both formats): [ceil(rows / 128)][ceil(scales per row / 4)][512 bytes], row r of a
// tile at 16 (r % 32) + 4 (r / 32 % 4), its four scales side by side: the image tcgen05.cp
// 32x128b takes into tensor memory. Scales past the end of K are zero bytes; rows past the last
// are left as they were (they only reach output rows that are not stored).
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "quantize_b.cuh"
#include "sm100.cuh"

namespace bd {

enum : int { kNvfp4 = 0, kMxfp4 = 1 };
enum : int { kInF32 = 0, kInBf16 = 1, kInF16 = 2 };

constexpr float kFp4RowMax = 2688.0f;  // 448 * 6

// Offset of scale s of row r in the tiles, `words` tiles (of four scales) per 128 rows.
__host__ __device__ __forceinline__ int64_t sf_tile_offset(int64_t r, int s, int words) {
  return ((r >> 7) * words + (s >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (s & 3);
}

// 16 consecutive elements as loaded.
template <int kIn>
struct Raw16 {
  static constexpr int kWords = kIn == kInF32 ? 16 : 8;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* x, int64_t elem) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) +
                                                    elem * (kIn == kInF32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 q = __ldg(p + i);
      w[4 * i] = q.x;
      w[4 * i + 1] = q.y;
      w[4 * i + 2] = q.z;
      w[4 * i + 3] = q.w;
    }
  }
  __device__ __forceinline__ float get(int j) const {  // j a constant after unrolling
    if constexpr (kIn == kInF32) return __uint_as_float(w[j]);
    else if constexpr (kIn == kInBf16)
      return __uint_as_float((j & 1) ? (w[j >> 1] & 0xFFFF0000u) : (w[j >> 1] << 16));
    else
      return __half2float(__ushort_as_half(
          static_cast<unsigned short>((j & 1) ? (w[j >> 1] >> 16) : (w[j >> 1] & 0xFFFFu))));
  }
  // bits of the largest magnitude (NaN above Inf above every finite value)
  __device__ __forceinline__ uint32_t amax_bits() const {
    if constexpr (kIn == kInF32) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) m = max(m, w[j] & 0x7FFFFFFFu);
      return m;
    } else {
      // two 16-bit patterns at a time: magnitudes order as unsigned integers
      uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
      for (int j = 1; j < 8; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
      const uint32_t b = max(m >> 16, m & 0xFFFFu);
      if constexpr (kIn == kInBf16) return b << 16;
      else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(b))));
    }
  }
};

// Four codes bytes of eight scaled elements, sign kept on non-zero magnitudes only.
__device__ __forceinline__ uint32_t e2m1_pack8(const float (&y)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  // a nibble's magnitude + 7 has bit 3 set exactly when it is not 0
  return w & ((((w & 0x77777777u) + 0x77777777u) & 0x88888888u) | 0x77777777u);
}

// 16 elements times r -> 8 code bytes. The conversion rounds ties to even, the rule to the lower
// magnitude, so a product that is a tie (its low 21 mantissa bits are zero) is made a little smaller.
// kLow: r is already 2^-20 too small, which does it for 16-bit elements and a power of two: a product
// has at most 11 significant bits, so it is a tie or at least 2^-11 of itself away from one.
template <int kIn, bool kLow>
__device__ __forceinline__ uint2 e2m1_encode16(const Raw16<kIn>& x, float r) {
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = __fmul_rn(x.get(8 * h + j), r);
      if (!kLow && (__float_as_uint(y[j]) & 0x1FFFFFu) == 0) y[j] = __fmul_rn(y[j], 0.99999994f);  // 1 - 2^-24
    }
    o[h] = e2m1_pack8(y);
  }
  return make_uint2(o[0], o[1]);
}

// Block exponent of MXFP4 from the bits of a finite amax: 6 * 2^e = 1.5 * 2^(e+2).
__device__ __forceinline__ int mxfp4_block_exp(uint32_t amax_bits) {
  if (amax_bits == 0u) return 0;
  const int E = static_cast<int>(amax_bits >> 23) - 127;
  return max(-40, min(40, E - 2 + ((amax_bits & 0x7FFFFFu) > 0x400000u ? 1 : 0)));
}

struct QuantFp4Params {
  const void* x;
  uint8_t* codes;
  uint8_t* scales;        // natural (M, K / block), may be null
  uint8_t* scales_tiled;  // tiles, may be null
  float* row_scale;       // (M,), NVFP4
  int M, K, words;
  int release;            // lets the next grid start early: the outputs are activations, not weights
  uint32_t* err;
};

// Quantiser. G threads share a row: a warp (eight to a CTA, no barriers), or a CTA of four or eight
// warps, their maxima meeting in shared memory; kKeep pieces of each thread are in flight. A thread takes
// 16-element pieces t, t + G, ..., keeps the first kKeep of them in registers between the maximum and the
// codes, and reads the rest of a long row twice (the second time from L2). Measured: 4099 x 14336 fp32 to
// MXFP4 47 us (5.6 TB/s), 8192 x 14336 bf16 to MXFP4 60 us (5.0 TB/s), 8192 x 4096 bf16 to NVFP4 28 us
// (3.1 TB/s: two divisions a block and the row's maximum first); 57 % of the issue slots, the integer pipe
// 60 % busy. Few rows are bound by the launch.
__host__ __device__ constexpr int q4_threads(int G) { return G == 32 ? 256 : G; }

template <int kIn, int kFmt, int G>
__global__ void __launch_bounds__(q4_threads(G), (kIn == kInF32 ? 2 : 3) * 256 / q4_threads(G))
    quantize_fp4_kernel(const QuantFp4Params p) {
  constexpr int kKeep = 4, kQ4Threads = q4_threads(G);
  constexpr bool kLow = kFmt == kMxfp4 && kIn != kInF32;
  __shared__ uint32_t part[2][kQ4Threads / 32];
  const int sub = threadIdx.x / G, t = threadIdx.x % G;
  const int pieces = p.K / 16;
  const int pieces_pad = (pieces + 7) & ~7;  // whole groups of eight: lanes past the end pad tiles
  // In this order: a W4A4 GEMM behind this grid may load weights before it waits, and they may be the
  // output of the grid before this one. Where this grid's own output may be weights it releases nothing: the
  // launch behind it may start the one after, which may stream weights early (weights_static is a promise
  // about the launch just before).
  grid_dep_wait();
  if (p.release) grid_dep_launch_dependents();
  bool bad = false;
  int flip = 0;
  for (int64_t m0 = static_cast<int64_t>(blockIdx.x) * (kQ4Threads / G); m0 < p.M;
       m0 += static_cast<int64_t>(gridDim.x) * (kQ4Threads / G)) {
    const int64_t m = m0 + sub;
    const bool row_ok = m < p.M;
    const int64_t e0 = m * p.K;
    Raw16<kIn> keep[kKeep];
    auto fetch = [&](int c0) {
#pragma unroll
      for (int u = 0; u < kKeep; ++u)
        if (row_ok && c0 + u * G < pieces)
          keep[u].load(p.x, e0 + static_cast<int64_t>(c0 + u * G) * 16);
    };
    float inv = 1.0f;
    if constexpr (kFmt == kNvfp4) {
      // the row's maximum, last pieces first: the first kKeep stay in registers
      uint32_t am = 0;
      for (int c0 = (pieces - 1) / (kKeep * G) * (kKeep * G) + t; c0 >= 0; c0 -= kKeep * G) {
        fetch(c0);
#pragma unroll
        for (int u = 0; u < kKeep; ++u)
          if (row_ok && c0 + u * G < pieces) am = max(am, keep[u].amax_bits());
      }
      am = __reduce_max_sync(0xFFFFFFFFu, am);
      if constexpr (G > 32) {
        // two sets of slots in turn: a warp of the next row cannot overwrite what a slower warp
        // of this one still reads
        if ((threadIdx.x & 31) == 0) part[flip][threadIdx.x >> 5] = am;
        __syncthreads();
        am = 0;
#pragma unroll
        for (int i = 0; i < G / 32; ++i) am = max(am, part[flip][i]);
        flip ^= 1;
      }
      bad |= am >= 0x7F800000u;
      const float s =
          am == 0u ? 1.0f
                   : fmaxf(__fdiv_rn(__uint_as_float(am), kFp4RowMax), 7.52316385e-37f);  // 2^-120
      inv = __frcp_rn(s);
      if (row_ok && t == 0) p.row_scale[m] = s;
    } else {
      fetch(t);
    }
    if (!row_ok) continue;  // whole warps (G is a multiple of 32)
    // Piece c of the row. Lanes of a group of eight pieces come together (pieces_pad and G are
    // multiples of eight, a warp's lanes hold consecutive pieces).
    const uint32_t group = 0xFFu << (threadIdx.x & 24);
    auto encode = [&](int c, const Raw16<kIn>& r) {
      const bool ok = c < pieces;
      uint32_t am = ok ? r.amax_bits() : 0u;
      uint32_t byte;
      float mul;
      if constexpr (kFmt == kNvfp4) {
        const float B = nvfp4_block_scale(__fmul_rn(__uint_as_float(am), inv), byte);
        mul = __fdiv_rn(inv, B);
      } else {
        am = max(am, __shfl_xor_sync(group, am, 1));
        bad |= am >= 0x7F800000u;
        const int e = mxfp4_block_exp(am);
        byte = static_cast<uint32_t>(e + 127);
        mul = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        if (kLow) mul *= 0.99999905f;  // 1 - 2^-20
      }
      if (!ok) byte = 0;
      if (ok)
        *reinterpret_cast<uint2*>(p.codes + (e0 >> 1) + static_cast<int64_t>(c) * 8) =
            e2m1_encode16<kIn, kLow>(r, mul);
      if constexpr (kFmt == kNvfp4) {
        if (p.scales != nullptr && ok) p.scales[m * pieces + c] = static_cast<uint8_t>(byte);
        if (p.scales_tiled != nullptr) {
          uint32_t w = byte << (8 * (c & 3));
          w |= __shfl_xor_sync(group, w, 1);
          w |= __shfl_xor_sync(group, w, 2);
          if ((c & 3) == 0 && (c >> 2) < p.words)
            *reinterpret_cast<uint32_t*>(p.scales_tiled + sf_tile_offset(m, c, p.words)) = w;
        }
      } else {
        if (p.scales != nullptr && ok && (c & 1) == 0)
          p.scales[m * (pieces / 2) + c / 2] = static_cast<uint8_t>(byte);
        if (p.scales_tiled != nullptr) {
          uint32_t w = byte << (8 * ((c >> 1) & 3));
          w |= __shfl_xor_sync(group, w, 2);
          w |= __shfl_xor_sync(group, w, 4);
          if ((c & 7) == 0)
            *reinterpret_cast<uint32_t*>(p.scales_tiled + sf_tile_offset(m, c / 2, p.words)) = w;
        }
      }
    };
    for (int c0 = t; c0 < pieces_pad; c0 += kKeep * G) {
      if (c0 != t) fetch(c0);
#pragma unroll
      for (int u = 0; u < kKeep; ++u)
        if (c0 + u * G < pieces_pad) encode(c0 + u * G, keep[u]);
    }
  }
  if (bad) atomicOr(p.err, kErrNonFinite);
}

// Natural scale bytes (rows, S) -> tiles; one thread per four scales, zeros past S.
__global__ void __launch_bounds__(256) tile_scales_kernel(const uint8_t* __restrict__ scales,
                                                          uint8_t* __restrict__ tiled, int rows,
                                                          int S, int words) {
  const int64_t total = static_cast<int64_t>(rows) * words;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / words;
    const int s = static_cast<int>(i % words) * 4;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (s + j < S) w |= static_cast<uint32_t>(scales[r * S + s + j]) << (8 * j);
    *reinterpret_cast<uint32_t*>(tiled + sf_tile_offset(r, s, words)) = w;
  }
}

// E2M1 nibble -> float.
__device__ __forceinline__ float e2m1_value(uint32_t n) {
  // magnitude index i: i / 2 below 2, else (1 + (i & 1) / 2) * 2^(i / 2 - 1)
  const uint32_t i = n & 7u;
  const uint32_t bits = i < 2 ? (i != 0u ? 0x3F000000u : 0u) : ((i + 252u) << 22);
  return __uint_as_float(bits | ((n & 8u) << 28));
}

__device__ __forceinline__ float e4m3_value(uint32_t b) {
  const uint32_t e = (b >> 3) & 15u, m = b & 7u;
  const float v = e != 0u ? __uint_as_float(((e + 120u) << 23) | (m << 20))
                          : static_cast<float>(m) * 0.001953125f;  // m * 2^-9
  return (b & 0x7Fu) == 0x7Fu ? __uint_as_float(0x7FC00000u) : ((b & 0x80u) ? -v : v);
}

__device__ __forceinline__ float e8m0_value(uint32_t b) {
  if (b == 0xFFu) return __uint_as_float(0x7FC00000u);
  return b != 0u ? __uint_as_float(b << 23) : __uint_as_float(0x00400000u);  // 2^-127
}

// Dequantiser: out (M, K) = (code * block scale) * (row scale * tensor scale), the first product
// exact. G threads share a row, each turn 16 bytes of output a thread (side by side); bound by the
// bytes written (4099 x 14336 to fp32: 52 us, 5.1 TB/s).
template <int kFmt, int kOut, int G>
__global__ void __launch_bounds__(256)
    dequantize_fp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ tiled,
                          const float* __restrict__ row_scale, float tensor_scale,
                          uint8_t* __restrict__ out, int M, int K, int words) {
  constexpr int kElems = kOut == 2 ? 4 : 8;      // per thread and turn
  constexpr int kPer = (kFmt == kNvfp4 ? 16 : 32) / kElems;  // threads per block scale
  constexpr int kTurns = 4;
  const int t = threadIdx.x % G, groups = K / kElems;
  grid_dep_wait();
  for (int64_t m = static_cast<int64_t>(blockIdx.x) * (256 / G) + threadIdx.x / G; m < M;
       m += static_cast<int64_t>(gridDim.x) * (256 / G)) {
    const float s = row_scale != nullptr ? __fmul_rn(row_scale[m], tensor_scale) : tensor_scale;
    const uint8_t* src = codes + m * (K / 2);
    const int64_t tile = sf_tile_offset(m, 0, words);
    uint8_t* dst = out + m * K * (16 / kElems);
    for (int g0 = t; g0 < groups; g0 += kTurns * G) {
      uint32_t q[kTurns], b[kTurns];
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        const int g = g0 + u * G;
        if (g < groups) {
          q[u] = kElems == 8 ? reinterpret_cast<const uint32_t*>(src)[g]
                             : reinterpret_cast<const uint16_t*>(src)[g];
          const int sc = g / kPer;
          b[u] = tiled[tile + static_cast<int64_t>(sc >> 2) * 512 + (sc & 3)];
        }
      }
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        const int g = g0 + u * G;
        if (g >= groups) break;
        const float sc = kFmt == kNvfp4 ? e4m3_value(b[u]) : e8m0_value(b[u]);
        float v[kElems];
#pragma unroll
        for (int j = 0; j < kElems; ++j)
          v[j] = __fmul_rn(__fmul_rn(e2m1_value((q[u] >> (4 * j)) & 15u), sc), s);
        uint4 w;
        if constexpr (kOut == 2) {
          w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                         __float_as_uint(v[3]));
        } else {
          uint32_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kOut == 0) {
              const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
              h[j] = *reinterpret_cast<const uint32_t*>(&x);
            } else {
              const __half2 x = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
              h[j] = *reinterpret_cast<const uint32_t*>(&x);
            }
          }
          w = make_uint4(h[0], h[1], h[2], h[3]);
        }
        __stcs(reinterpret_cast<uint4*>(dst) + g, w);
      }
    }
  }
}

}  // namespace bd
