// Launch helpers of the generation kernels.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"

namespace mnb {

// A kernel whose next one in the stream was launched by launch_after(): the next may start from here on.
MNB_DEVICE void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// A kernel launched by launch_after(): past this point the kernel before it has ended and its results are there.
MNB_DEVICE void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Starts while the kernel before it in the stream still runs, as far as there is room on the SMs.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), int blocks, int threads, int bytes, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A kernel's limit of dynamic shared memory on each device, raised when a launch needs more than any before, and then to
// all that the kernel can have (`most`): every call sets the same value, so that calls from several threads agree.
struct SharedMemory {
  static constexpr int kDevices = 64;
  std::atomic<int> limit[kDevices] = {};
  cudaError_t at_least(const void* kernel, int bytes, int most = 227 * 1024 - 4096) {
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    if (dev < kDevices && bytes <= limit[dev].load(std::memory_order_acquire)) return cudaSuccess;
    if (most < bytes) most = bytes;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess && dev < kDevices) limit[dev].store(most, std::memory_order_release);
    return e;
  }
};

}  // namespace mnb
