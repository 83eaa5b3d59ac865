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

}  // namespace attnres_b200
