// The two 16-bit floating types the windowed attention, rotary and cache operators take, behind one
// set of conversions.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace aici {

template <typename T>
struct Half16;

template <>
struct Half16<__nv_bfloat16> {
  static constexpr int kDtype = AICI_DTYPE_BF16;
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
};

template <>
struct Half16<__half> {
  static constexpr int kDtype = AICI_DTYPE_F16;
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
};

// Calls f with a value of the type that `dtype` (AICI_DTYPE_BF16 or AICI_DTYPE_F16) names.
template <typename F>
inline char *with_half_type(int dtype, F f) {
  return dtype == AICI_DTYPE_F16 ? f(__half()) : f(__nv_bfloat16());
}

}  // namespace aici
