// Eight-bit pages: e4m3 codes with one fp32 scale for each page and head.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "grs_common.cuh"

namespace grs {

// The smallest power of two s with amax <= 448 s (448 is e4m3's largest value), kept
// within 2^-118 .. 2^119 so that s and 1 / s are normal.  Powers of two: codes move
// from one scale to another exactly, but for those that become subnormal.
__device__ __forceinline__ float e4m3_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);   // 448 = 1.75 * 2^8
  return __uint_as_float((uint32_t)(min(max(e, -118), 119) + 127) << 23);
}

// What is not finite cannot be held and becomes NaN (the conversion alone would make
// 448 of an infinity).
__device__ __forceinline__ float e4m3_checked(float x) {
  return fabsf(x) <= 3.402823466e38f ? x : __uint_as_float(0x7fffffffu);
}
__device__ __forceinline__ uint8_t to_e4m3(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(e4m3_checked(x), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float from_e4m3(uint8_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

}  // namespace grs
