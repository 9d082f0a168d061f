// Host helpers shared by the translation units of the 4-bit cache.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gfx906_b200_cache4.h"

// Defined in attn_fwd_sm100.cu: the checks of the current device (sm_100, SM
// count under the process-wide cap) and the thread's last status.
extern "C" int gfx906_b200_internal_device(int* num_sms);
extern "C" int gfx906_b200_internal_set_last_error(int status);
extern "C" unsigned long long gfx906_b200_internal_timeout_ns(void);

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

inline int done(int status) { return gfx906_b200_internal_set_last_error(status); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool head_dim_ok(int D) { return D == 64 || D == 128; }

}  // namespace c4
