// Rotary positions: pair i of a head's first 2 * pairs elements is turned by the
// angle position * f_i.  Shared by rotary.cu and token_cache.cu.
//
// Angles are held in turns, a pair's step as a 128-bit fixed-point fraction: position
// * step is taken modulo whole turns in integers, so the angle of a far position is
// as exact as that of a near one, for every 64-bit position (fp32 angles are off by
// 0.06 rad at position 10^6).  Only the reduced angle, at most pi / 4, becomes a
// float.
#pragma once

#include <type_traits>

#include "grs_common.cuh"

namespace grs {

// f / (2 pi) in turns, modulo 1, in units of 2^-64 (hi) and 2^-128 (lo).  1 / (2 pi)
// is the sum of two doubles: the fraction is exact to 2^-108 of a radian's turn.
struct RotaryStep {
  uint64_t hi, lo;
};
__device__ __forceinline__ RotaryStep rotary_step(double f) {
  constexpr double hi = 0x1.45f306dc9c883p-3, lo = -0x1.6b01ec5417056p-57;
  const double t = f * hi;
  const double rest = fma(f, hi, -t) + f * lo;
  const double a = (t - rint(t)) * 0x1p64, whole = rint(a);     // both exact
  const double b = (a - whole) + rest * 0x1p64, low = floor(b);
  return {(uint64_t)__double2ll_rn(whole) + (uint64_t)__double2ll_rn(low),
          __double2ull_rz((b - low) * 0x1p64)};
}
// The phase of a position, a fraction of a turn in units of 2^-64.
__device__ __forceinline__ uint64_t rotary_phase(int64_t position, RotaryStep step) {
  const uint64_t p = (uint64_t)position;
  return p * step.hi + __umul64hi(p, step.lo) - (position < 0 ? step.lo : 0);
}

// (cos, sin) of a phase.  The nearest quarter turn is taken off; the rest z, |z| <=
// pi / 4, goes through the Taylor series up to z^9 and z^10, whose next terms are
// below 1.8e-9 and 1.2e-10.
__device__ __forceinline__ float2 rotary_cos_sin(uint64_t phase) {
  const uint32_t turn = (uint32_t)((phase + 0x80000000ull) >> 32);
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float z = (float)(int32_t)(turn - (quarter << 30)) * 1.46291808e-9f;   // 2 pi / 2^32
  const float y = z * z;
  float s = fmaf(y, 2.75573192e-6f, -1.98412698e-4f);
  s = fmaf(y, s, 8.33333333e-3f);
  s = fmaf(y, s, -1.66666667e-1f);
  s = fmaf(y * z, s, z);
  float c = fmaf(y, -2.75573192e-7f, 2.48015873e-5f);
  c = fmaf(y, c, -1.38888889e-3f);
  c = fmaf(y, c, 4.16666667e-2f);
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.f);
  const float x = quarter & 1 ? -s : c, w = quarter & 1 ? c : s;
  return quarter & 2 ? make_float2(-x, -w) : make_float2(x, w);
}

// kVec consecutive elements, moved as one word.
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) RotaryPiece {
  T e[kVec];
};

// A head as units of one thread: a piece of each element of kVec pairs (halves, or
// kVec == 1), or one piece that holds whole pairs; the elements behind the pairs
// are pieces of their own.
template <int kVec, bool kInter>
struct RotaryUnits {
  static constexpr bool kTwo = !kInter || kVec == 1;
  static __host__ __device__ int count(int width, int pairs) {
    return kTwo ? (width - pairs) / kVec : width / kVec;
  }
  static __host__ __device__ bool takes(int width, int pairs) {
    return width % kVec == 0 && (kTwo ? pairs : 2 * pairs) % kVec == 0;
  }
  int a, b, pair;                           // places of the pieces, first pair; pair < 0: kept
  __device__ __forceinline__ RotaryUnits(int u, int pairs) {
    if constexpr (kTwo) {
      const bool turned = u * kVec < pairs;
      a = !turned ? pairs + u * kVec : kInter ? 2 * u : u * kVec;
      b = kInter ? a + 1 : a + pairs;
      pair = turned ? u * kVec : -1;
    } else {
      a = u * kVec;
      b = a;
      pair = a < 2 * pairs ? a / 2 : -1;
    }
  }
  __device__ __forceinline__ bool two() const { return kTwo && pair >= 0; }
};

// Turns the unit's pieces by its pairs' (cos, sin).
template <typename T, int kVec, bool kInter>
__device__ __forceinline__ void rotary_turn(const float2* cs, float (&x)[kVec], float (&y)[kVec]) {
  if constexpr (RotaryUnits<kVec, kInter>::kTwo) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float2 t = cs[i];
      const float a = x[i], b = y[i];
      x[i] = fmaf(a, t.x, -b * t.y);
      y[i] = fmaf(a, t.y, b * t.x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      const float2 t = cs[i];
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = fmaf(a, t.x, -b * t.y);
      x[2 * i + 1] = fmaf(a, t.y, b * t.x);
    }
  }
}

// The widest piece that `takes` the layout: calls f with its width (16 bytes, 8, or one
// element) and whether pairs lie side by side.
template <typename T, typename F>
static int rotary_dispatch(int width, int pairs, bool interleaved, int alignment, F f) {
  constexpr int kWide = 16 / sizeof(T), kHalf = kWide / 2;
  const auto with = [&](auto inter) {
    constexpr bool kInter = decltype(inter)::value;
    if (alignment % 16 == 0 && RotaryUnits<kWide, kInter>::takes(width, pairs))
      return f(std::integral_constant<int, kWide>{}, inter);
    if (alignment % 8 == 0 && RotaryUnits<kHalf, kInter>::takes(width, pairs))
      return f(std::integral_constant<int, kHalf>{}, inter);
    return f(std::integral_constant<int, 1>{}, inter);
  };
  return interleaved ? with(std::true_type{}) : with(std::false_type{});
}

// The largest power of two, up to 16, that divides an address and byte strides.
static inline int common_alignment(const void* at, int64_t s0 = 0, int64_t s1 = 0, int64_t s2 = 0) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(at) | (uint64_t)s0 | (uint64_t)s1 |
                        (uint64_t)s2 | 16;
  return (int)(bits & -bits);
}

}  // namespace grs
