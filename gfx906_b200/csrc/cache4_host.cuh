// Host helpers shared by the translation units of the 4-bit cache.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/gfx906_b200_cache4.h"

// Defined in attn_fwd_sm100.cu: the checks of the current device (sm_100, SM
// count under the process-wide cap) and the thread's last status.
extern "C" int gfx906_b200_internal_device(int* num_sms);
extern "C" int gfx906_b200_internal_set_last_error(int status);
extern "C" unsigned long long gfx906_b200_internal_timeout_ns(void);
extern "C" unsigned long long gfx906_b200_internal_next_epoch(void);  // unique per launch, 56 bits

namespace c4 {

// Launch that may begin while the previous kernel on the stream ends; every
// kernel launched so waits (griddepcontrol.wait) before its first global access.
template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? GFX906_B200_OK : GFX906_B200_ECUDA;
}

// Raises a kernel's limit of dynamic shared memory once per device.
class SmemAttribute {
 public:
  template <typename K>
  bool set(K* kernel, int bytes) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    const unsigned long long bit = 1ull << dev;
    if (set_.load(std::memory_order_acquire) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    set_.fetch_or(bit, std::memory_order_release);
    return true;
  }

 private:
  std::atomic<unsigned long long> set_{0};
};

inline int done(int status) { return gfx906_b200_internal_set_last_error(status); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool head_dim_ok(int D) { return D == 64 || D == 128; }

}  // namespace c4
