// Host side of kernel launches.
#pragma once
#include <atomic>
#include <cuda_runtime.h>

extern "C" void msb_set_error(const char* fmt, ...);

namespace msb {
// Lets `kern` be launched with `bytes` of dynamic shared memory on the current device.  The limit belongs to the device, so it is
// stated once per device of the process; `stated` is the launcher's own record (a bit per device, static).
inline int allow_smem(const void* kern, int bytes, const char* what, std::atomic<unsigned long long>& stated) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;      // devices past the record are told every time
  if (e == cudaSuccess && (stated.load(std::memory_order_relaxed) & bit)) return 0;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    msb_set_error("%s: cannot set %d bytes of dynamic shared memory: %s", what, bytes, cudaGetErrorString(e));
    return 1;
  }
  stated.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

#ifdef __CUDACC__
// Launch of a kernel that begins while the one before it on the stream ends: its blocks are placed and set up early and wait in
// `after_previous()`, which every thread of such a kernel calls before it touches memory that an earlier kernel writes or reads.  What
// earlier kernels of the same chain wrote must not be read through `const __restrict__` pointers (the compiler may move such loads).
// The first kernel of a chain is launched the ordinary way.
template <typename... P, typename... A>
inline cudaError_t launch_after(void (*kern)(P...), dim3 grid, unsigned block, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid; c.blockDim = dim3(block); c.dynamicSmemBytes = smem; c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at; c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kern, P(args)...);
}
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
#endif
}  // namespace msb
