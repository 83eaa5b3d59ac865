// Host-side helpers and the element types shared by the C-ABI translation units.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/attnres_b200.h"

namespace attnres_b200 {

inline int sm_count(int device, int* out) {
  // Queried per call: the attribute lookup is a cached driver read and keeps
  // the library free of mutable global state.
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      sms < 1) {
    cudaGetLastError();
    return ATTNRES_B200_ERR_CUDA;
  }
  *out = sms;
  return ATTNRES_B200_OK;
}

inline int current_device(int* device) {
  if (cudaGetDevice(device) != cudaSuccess) {
    cudaGetLastError();
    return ATTNRES_B200_ERR_CUDA;
  }
  return ATTNRES_B200_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

inline int launched() {
  return cudaGetLastError() == cudaSuccess ? ATTNRES_B200_OK : ATTNRES_B200_ERR_CUDA;
}

inline bool type_ok(int32_t type) {
  return type == ATTNRES_B200_BF16 || type == ATTNRES_B200_FP16 || type == ATTNRES_B200_FP32;
}

inline int type_bytes(int32_t type) { return type == ATTNRES_B200_FP32 ? 4 : 2; }

// Whether a pointer sits on a boundary of its own element type.
inline bool aligned_type(const void* p, int32_t type) {
  return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(type_bytes(type) - 1)) == 0;
}

// A launch that may begin before the kernel in front of it has ended: once all of that kernel's CTAs
// have called start_next_kernel() or are done.  The launched kernel calls wait_for_previous_kernel()
// before it touches anything the kernels in front of it read or write.
template <typename... Parameters, typename... Arguments>
int launch_behind(void (*kernel)(Parameters...), int64_t grid, int threads, uint32_t smem, bool behind,
                  cudaStream_t stream, const Arguments&... arguments) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)grid);
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = behind ? 1 : 0;
  if (cudaLaunchKernelEx(&config, kernel, Parameters(arguments)...) != cudaSuccess) {
    cudaGetLastError();
    return ATTNRES_B200_ERR_CUDA;
  }
  return ATTNRES_B200_OK;
}

__device__ __forceinline__ void start_next_kernel() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous_kernel() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace attnres_b200
