// sp24_host.cuh — host-side plumbing shared by the library's translation
// units: error macro, device table, TMA tensor-map encoding, kernel attributes
// and launches.  Definitions that own state live in sp24_api.cu.
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>
#include <utility>

#include "../../include/sp24.h"

#define SP24_CUDA_TRY(expr)                  \
  do {                                       \
    cudaError_t e__ = (expr);                \
    if (e__ != cudaSuccess) {                \
      (void)cudaGetLastError();              \
      return SP24_ERR_CUDA;                  \
    }                                        \
  } while (0)

namespace sp24host {

constexpr int kMaxDevices = 64;
constexpr unsigned long long kDefaultTimeoutNs = 1000000000ull;  // 1 s per bounded wait

inline cudaStream_t as_stream(sp24_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }
inline size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }
// 128-row blocks of the tcgen05 metadata image, padded to an even count so a
// CTA pair's second half always has an atom to load.
inline int meta_mblocks(int m) { return ((m + 127) / 128 + 1) / 2 * 2; }
inline int meta_katoms(int k) { return (k + 127) / 128; }

struct DeviceInfo {
  int sm_count = 0;
  int* status_word = nullptr;
  bool ok = false;
};

// The current device's entry; SP24_ERR_ARCH when it is no sm_100 part.
sp24_status device_info(DeviceInfo** out);

// 2-D TMA tensor map (inner extent contiguous).
sp24_status encode_2d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, uint64_t inner,
                      uint64_t outer, uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer,
                      CUtensorMapSwizzle sw);

extern std::mutex g_attr_mu;

// Sets a kernel's function attributes (dynamic shared memory, and the
// non-portable cluster size when asked) once per device.  `done` is the
// calling launcher's own per-device flag array; the first calls on a device
// from several host threads serialise on the mutex.
template <typename Kern>
sp24_status ensure_kernel_attrs(Kern kern, std::atomic<bool> (&done)[kMaxDevices], int smem,
                                bool nonportable_cluster = false) {
  int dev = 0;
  SP24_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return SP24_ERR_ARG;
  if (done[dev].load(std::memory_order_acquire)) return SP24_OK;
  std::lock_guard<std::mutex> lk(g_attr_mu);
  if (done[dev].load(std::memory_order_relaxed)) return SP24_OK;
  SP24_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (nonportable_cluster)
    SP24_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  done[dev].store(true, std::memory_order_release);
  return SP24_OK;
}

// GEMM launches carry programmatic stream serialization: the kernel may be
// scheduled while the previous kernel of the stream finishes, runs its
// prologue (barriers, TMEM allocation, tensor-map prefetch), and its TMA
// producers wait for the previous grid (griddepcontrol.wait) before the
// first load.  pdl = false launches without the attribute.
template <typename... KArgs, typename... Args>
sp24_status launch_gemm_kernel(void (*kern)(KArgs...), unsigned grid, unsigned block, size_t smem,
                               cudaStream_t stream, unsigned cluster, bool pdl, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned na = 0;
  if (cluster > 0) {   // run-time cluster shape; 0 = none (or the kernel's __cluster_dims__)
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = cluster;
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    ++na;
  }
  if (pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  SP24_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...));
  return SP24_OK;
}

}  // namespace sp24host
