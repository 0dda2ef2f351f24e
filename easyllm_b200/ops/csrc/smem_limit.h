// Dynamic shared memory above 48 KB, asked for once for each kernel and device.
//
// The limit is an attribute of a kernel on the device that is current when it is set.  A process may use several devices, and the launchers
// make a tensor's own the current one, so what was set is remembered for each.  Host code only.
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <mutex>

namespace ell {

struct SmemLimit {                // of one kernel; a static object of its launcher
  static constexpr int kDevices = 64;
  std::atomic<int> bytes[kDevices] = {};
  std::mutex setting;
};

// The kernel may be launched on the current device with `bytes` of dynamic shared memory, or an error code.
inline int allow_smem_of(const void* kern, int bytes, SmemLimit& had) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= SmemLimit::kDevices) return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (had.bytes[dev].load(std::memory_order_acquire) >= bytes) return 0;
  std::lock_guard<std::mutex> lock(had.setting);       // of two sizes that are set at once the larger one stays
  if (had.bytes[dev].load(std::memory_order_relaxed) >= bytes) return 0;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) had.bytes[dev].store(bytes, std::memory_order_release);
  return (int)e;
}
template <typename... P>
inline int allow_smem(void (*kern)(P...), int bytes, SmemLimit& had) {
  return allow_smem_of(reinterpret_cast<const void*>(kern), bytes, had);
}

}  // namespace ell
