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

// Eight elements of one row as they lie in memory (the upper half is used by FP32 only), so that
// loads can be issued ahead of the conversions.
struct Raw8 {
  uint4 a, b;
};

// With VECTOR the eight are consecutive from `index`, 16-byte aligned and all valid.  Otherwise
// element e is `index + e * step` (so that neighbouring lanes read neighbouring elements), and
// only the first `count` exist.
template <bool VECTOR>
__device__ __forceinline__ Raw8 load_raw8(const void* base, int type, int64_t index, int step,
                                          int count) {
  Raw8 r;
  r.a = make_uint4(0u, 0u, 0u, 0u);
  r.b = r.a;
  if constexpr (VECTOR) {
    if (type == ATTNRES_B200_FP32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + index);
      r.a = __ldg(p);
      r.b = __ldg(p + 1);
    } else {
      r.a = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(base) + index));
    }
  } else {
    uint32_t w[8];
    if (type == ATTNRES_B200_FP32) {
      const uint32_t* p = static_cast<const uint32_t*>(base) + index;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = e < count ? __ldg(p + e * step) : 0u;
      r.a = make_uint4(w[0], w[1], w[2], w[3]);
      r.b = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
      const unsigned short* p = static_cast<const unsigned short*>(base) + index;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = e < count ? (uint32_t)__ldg(p + e * step) : 0u;
      r.a = make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16),
                       w[6] | (w[7] << 16));
    }
  }
  return r;
}

__device__ __forceinline__ void unpack_raw8(const Raw8& r, int type, float* f) {
  if (type == ATTNRES_B200_FP32) {
    f[0] = __uint_as_float(r.a.x);
    f[1] = __uint_as_float(r.a.y);
    f[2] = __uint_as_float(r.a.z);
    f[3] = __uint_as_float(r.a.w);
    f[4] = __uint_as_float(r.b.x);
    f[5] = __uint_as_float(r.b.y);
    f[6] = __uint_as_float(r.b.z);
    f[7] = __uint_as_float(r.b.w);
  } else if (type == ATTNRES_B200_BF16) {
    unpack8(r.a, f);
  } else {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[2 * k] = v.x;
      f[2 * k + 1] = v.y;
    }
  }
}

template <bool VECTOR>
__device__ __forceinline__ void store8(void* base, int type, int64_t index, int step, int count,
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
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) store_typed(base, type, index + e * step, f[e]);
  }
}

}  // namespace attnres_b200
