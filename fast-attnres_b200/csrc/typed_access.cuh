// Element access for operators whose tensors may be BF16, FP16 or FP32: conversion of single
// elements, and eight consecutive elements at once when a runtime type code says which of the
// three they are (the branch is uniform over the grid and cheap beside the access itself).
#pragma once

#include "common.cuh"
#include "host_common.cuh"

namespace attnres_b200 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// One rounding to nearest even, as torch's own casts.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float load_typed(const void* base, int type, int64_t index) {
  if (type == ATTNRES_B200_FP32) return static_cast<const float*>(base)[index];
  if (type == ATTNRES_B200_BF16) return to_float(static_cast<const __nv_bfloat16*>(base)[index]);
  return to_float(static_cast<const __half*>(base)[index]);
}

__device__ __forceinline__ void store_typed(void* base, int type, int64_t index, float v) {
  if (type == ATTNRES_B200_FP32) static_cast<float*>(base)[index] = v;
  else if (type == ATTNRES_B200_BF16) static_cast<__nv_bfloat16*>(base)[index] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[index] = __float2half_rn(v);
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A lane's share of one row as it lies in memory: eight consecutive elements (VECTOR: 16-byte
// aligned and all valid), or E elements a step apart, so that neighbouring lanes read neighbouring
// elements, of which the first `count` exist.  Whether elements are 4 or 2 bytes wide is a template
// parameter (so that loads can be issued in batches, with no branch between them); which of the
// two 16-bit types they are only matters to the conversion and is a runtime code.
template <bool VECTOR, bool WIDE, int E = 8>
struct Share {
  static_assert(!VECTOR || E == 8, "a vector share is eight elements");
  static constexpr int kWords = !VECTOR ? E : WIDE ? 8 : 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const void* base, int64_t index, int step, int count) {
    if constexpr (VECTOR) {
      const char* p = static_cast<const char*>(base) + index * (WIDE ? 4 : 2);
      *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(p));
      if constexpr (WIDE) *reinterpret_cast<uint4*>(w + 4) = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    } else if constexpr (WIDE) {
      const uint32_t* p = static_cast<const uint32_t*>(base) + index;
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = e < count ? __ldg(p + e * step) : 0u;
    } else {
      const unsigned short* p = static_cast<const unsigned short*>(base) + index;
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = e < count ? (uint32_t)__ldg(p + e * step) : 0u;
    }
  }

  __device__ __forceinline__ void unpack(int type, float* f) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = __uint_as_float(w[e]);
    } else if constexpr (VECTOR) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        f[2 * k] = type == ATTNRES_B200_BF16 ? bf16x2_lo(w[k]) : h.x;
        f[2 * k + 1] = type == ATTNRES_B200_BF16 ? bf16x2_hi(w[k]) : h.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        f[e] = type == ATTNRES_B200_BF16 ? bf16_bits_to_float(w[e])
                                         : __half2float(__ushort_as_half((unsigned short)w[e]));
    }
  }
};

// Rounds and stores a share; `type` is the destination's.
template <bool VECTOR, int E = 8>
__device__ __forceinline__ void store_share(void* base, int type, int64_t index, int step, int count,
                                            const float* f) {
  if constexpr (VECTOR) {
    if (type == ATTNRES_B200_FP32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + index);
      p[0] = make_float4(f[0], f[1], f[2], f[3]);
      p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      uint4 v;
      if (type == ATTNRES_B200_BF16) {
        v = pack8(f);
      } else {
        v = make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]),
                       pack_half2(f[6], f[7]));
      }
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(base) + index) = v;
    }
  } else if (type == ATTNRES_B200_FP32) {
    float* p = static_cast<float*>(base) + index;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < count) p[e * step] = f[e];
  } else {
    unsigned short w[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      w[e] = type == ATTNRES_B200_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[e]))
                                       : __half_as_ushort(__float2half_rn(f[e]));
    unsigned short* p = static_cast<unsigned short*>(base) + index;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < count) p[e * step] = w[e];
  }
}

}  // namespace attnres_b200
