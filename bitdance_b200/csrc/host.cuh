// host.cuh -- host-side helpers shared by the translation units of the library: per-device
// facts, tensor maps, grid sizes (defined in bitdance.cu).
#pragma once
#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/bitdance_b200.h"

namespace bd {

constexpr int kMaxDevices = 64;

inline cudaStream_t as_stream(bd_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

inline bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// Per-device facts, computed once.
struct DeviceInfo {
  int sm_count = 0;
  bool is_sm100 = false;
  uint32_t* err = nullptr;
  bool ready = false;
};

// Facts of the current device: BD_OK, BD_ERR_ARCH when it is not an sm_100, BD_ERR_CUDA.
int device_info(DeviceInfo** out);

// 2-D tensor map of d1 rows of d0 elements, boxes of b1 rows x b0 elements, zero fill.
bool make_map_2d(CUtensorMap* m, CUtensorMapDataType dt, void* base, uint64_t d0, uint64_t d1,
                 uint64_t stride1_bytes, uint32_t b0, uint32_t b1, CUtensorMapSwizzle sw);

// Blocks for `work` items, per_block at a time, at most eight per SM.
int grid_for(int64_t work, int per_block, const DeviceInfo* d);

// Status of a launch (or of another runtime call) that returned e. A failed one leaves its error in the
// runtime's record as well: cleared here, so that no later call takes it for its own.
inline int launch_status(cudaError_t e) {
  if (e == cudaSuccess) return BD_OK;
  cudaGetLastError();
  return BD_ERR_CUDA;
}

}  // namespace bd
