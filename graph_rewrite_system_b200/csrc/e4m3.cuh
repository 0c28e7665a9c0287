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


// Two fp32 values to two codes, the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// Two codes times `ratio`, a power of two up to 1, in f16: exact for results that f16
// holds as normal numbers, and those that it does not are below 2^-14, which e4m3
// rounds to zero all the same.
__device__ __forceinline__ uint32_t e4m3x2_times(uint32_t codes, __half2 ratio) {
  uint32_t x;
  uint16_t y;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(x) : "h"((uint16_t)codes));
  const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&x), ratio);
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(y) : "r"(*reinterpret_cast<const uint32_t*>(&z)));
  return y;
}

// Four codes times any ratio, in fp32.
static __device__ __noinline__ uint32_t e4m3x4_times(uint32_t codes, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    out |= (uint32_t)to_e4m3(from_e4m3((uint8_t)(codes >> i)) * ratio) << i;
  return out;
}
// kVec values over a scale, stored as one word.  x * 0 + x * inverse: an infinity becomes
// NaN without a branch.
template <int kVec>
__device__ __forceinline__ void e4m3_store(uint8_t* at, const float (&x)[kVec], float inverse) {
  if constexpr (kVec == 1) {
    *at = (uint8_t)to_e4m3x2(fmaf(x[0], inverse, x[0] * 0.f), 0.f);
  } else {
    const uint64_t by = (uint64_t)__float_as_uint(inverse) << 32 | __float_as_uint(inverse);
    uint32_t w[(kVec + 3) / 4] = {};
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      uint64_t y = (uint64_t)__float_as_uint(x[i + 1]) << 32 | __float_as_uint(x[i]), z;
      asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(z) : "l"(y), "l"(0ull));
      asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(y) : "l"(y), "l"(by), "l"(z));
      w[i / 4] |= to_e4m3x2(__uint_as_float((uint32_t)y), __uint_as_float((uint32_t)(y >> 32)))
                  << 8 * (i % 4);
    }
    if constexpr (kVec == 2)
      *reinterpret_cast<uint16_t*>(at) = (uint16_t)w[0];
    else if constexpr (kVec == 4)
      *reinterpret_cast<uint32_t*>(at) = w[0];
    else
      *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
  }
}

}  // namespace grs
