// Host-side helpers shared by the C-ABI entry points: cached per-device
// properties and TMA tensor-map encoding through the driver entry point (so
// the library needs no link-time libcuda and loads on machines without a GPU).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>

namespace moe {

constexpr int kMaxDevices = 64;

struct DeviceInfo {
  int sm_count;
  int major;
  int minor;
};

// Device that is current on the calling thread and its cached properties.
int current_device_info(int* dev, DeviceInfo* info);

// cuTensorMapEncodeTiled with the given swizzle (128-byte by default), zero OOB
// fill, 256B L2 promotion.  strides_bytes has rank-1 entries (dimension 0 is
// contiguous).
int encode_tiled(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base,
                 const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                 CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B);

// Lets `kern` use `bytes` of dynamic shared memory on the current device, once per
// kernel and device (the attribute call costs about as much as a launch's share of it).
template <auto kern>
inline bool allow_shared_memory(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
  const uint64_t bit = uint64_t(1) << dev;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// MOE_B200_GEMM_KERNEL=1 selects the 1-SM kernels even for grids of two or more
// SMs (read once per process); the default is the CTA-pair kernels.
inline bool force_single_sm_kernel() {
  static const bool v = [] {
    const char* e = std::getenv("MOE_B200_GEMM_KERNEL");
    return e != nullptr && std::atoi(e) == 1;
  }();
  return v;
}

}  // namespace moe
