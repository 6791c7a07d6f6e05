// Host-side helpers that the library's translation units share: errors, device set-up, launches.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdlib>
#include <utility>

#define QGH_LOCAL __attribute__((visibility("hidden")))

namespace qgh {

// Keeps the message for qgemm_last_error() and returns -1.
QGH_LOCAL int fail(const char* fmt, ...);

// The set-up of the current device, once per device.
QGH_LOCAL int ensure_device(int* sm_count);

#define CUDA_OK(expr)                                                                          \
  do {                                                                                         \
    cudaError_t e_ = (expr);                                                                   \
    if (e_ != cudaSuccess) return qgh::fail("%s failed: %s", #expr, cudaGetErrorString(e_));   \
  } while (0)

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch `kernel` so that it may start while the kernel in front of it on the stream is still running
// (programmatic dependent launch); the kernel itself waits before it reads that kernel's results.
// QGEMM_PDL=0 falls back to plain stream order.  cluster > 1: in thread-block clusters of that many CTAs.
template <typename... KArgs, typename... Args>
int launch_pdl_clusters(void (*kernel)(KArgs...), int grid, int cluster, int threads, int smem, cudaStream_t s, Args&&... args) {
  static const int pdl = getenv("QGEMM_PDL") ? atoi(getenv("QGEMM_PDL")) : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
  return 0;
}
template <typename... KArgs, typename... Args>
int launch_pdl(void (*kernel)(KArgs...), int grid, int threads, int smem, cudaStream_t s, Args&&... args) {
  return launch_pdl_clusters(kernel, grid, 1, threads, smem, s, std::forward<Args>(args)...);
}

}  // namespace qgh
