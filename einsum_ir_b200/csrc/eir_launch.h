// Kernel launches of the library: every kernel is launched with programmatic
// stream serialisation (programmatic dependent launch), so its launch and
// prologue overlap the tail of the previous kernel in the stream. Each kernel
// calls pdl_wait() (eir_common.cuh) before its first global memory access and
// pdl_launch_dependents() once all of its CTAs are running. EIR_PDL=0 turns
// the attribute off (plain stream order).
#pragma once

#include <cuda_runtime.h>
#include <cstdlib>
#include <mutex>

namespace eir {

inline bool pdl_enabled() {
  static const bool on = [] {
    char const *v = std::getenv("EIR_PDL");
    return !(v != nullptr && v[0] == '0');
  }();
  return on;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                          cudaStream_t st, Args const &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Allows a kernel all the dynamic shared memory that its static words leave of a block's 227 KB, on the current
// device. The limit belongs to the kernel, not to a call: one that set it to its own size could lower it between
// another host thread's setting and launch, which is refused then. So it is set once, to the same value by all.
inline cudaError_t allow_all_smem(void const *kern) {
  struct Done {
    void const *kern;
    int dev;
  };
  static std::mutex mu;
  static Done done[1024];
  static int n = 0;  // (beyond the table's end a kernel's limit is set on every call)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  for (int i = 0; i < n; ++i)
    if (done[i].kern == kern && done[i].dev == dev) return cudaSuccess;
  cudaFuncAttributes fa;
  e = cudaFuncGetAttributes(&fa, kern);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)fa.sharedSizeBytes);
  if (e == cudaSuccess && n < 1024) done[n++] = Done{kern, dev};
  return e;
}

}  // namespace eir
