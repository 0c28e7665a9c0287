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
// A whole number from -2^63 to 2^63, modulo 2^64: half a turn, 2^63, is no int64.
__device__ __forceinline__ uint64_t rotary_units(double x) {
  return x < 0 ? (uint64_t)__double2ll_rn(x) : __double2ull_rn(x);
}
__device__ __forceinline__ RotaryStep rotary_step(double f) {
  constexpr double hi = 0x1.45f306dc9c883p-3, lo = -0x1.6b01ec5417056p-57;
  const double t = f * hi;
  double rest = fma(f, hi, -t) + f * lo;
  rest -= rint(rest);                       // whole turns of f from 2^53 on
  const double a = (t - rint(t)) * 0x1p64, whole = rint(a);     // both exact
  const double b = (a - whole) + rest * 0x1p64, low = floor(b);
  return {rotary_units(whole) + rotary_units(low), __double2ull_rz((b - low) * 0x1p64)};
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

// kVec consecutive elements, moved as one word and held as such.
template <typename T, int kVec>
struct RotaryPiece {
  static constexpr int kBytes = sizeof(T) * kVec;
  using Word = typename std::conditional<
      kBytes == 16, uint4, typename std::conditional<
      kBytes == 8, uint2, typename std::conditional<
      kBytes == 4, uint32_t, uint16_t>::type>::type>::type;
  Word word;
  __device__ __forceinline__ void clear() { word = Word(); }
  __device__ __forceinline__ void load(const T* at) { word = *reinterpret_cast<const Word*>(at); }
  __device__ __forceinline__ void store(T* at) const { *reinterpret_cast<Word*>(at) = word; }
  __device__ __forceinline__ void get(float (&x)[kVec]) const {
    if constexpr (kBytes < 4) {
      x[0] = __uint_as_float((uint32_t)word << 16);
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&word);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if constexpr (sizeof(T) == 4)
          x[i] = __uint_as_float(w[i]);
        else
          x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      }
    }
  }
  // The largest absolute value as its fp32 bits (not finite: 0x7f800000 and above, or
  // with `finite` left out).
  __device__ __forceinline__ uint32_t largest(bool finite) const {
    uint32_t top = 0;
    if constexpr (kBytes >= 4 && sizeof(T) == 2) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&word);
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) {
        uint32_t x = w[i] & 0x7fff7fffu;
        if (finite) {
          if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
          if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
        }
        top = __vmaxu2(top, x);
      }
      return max(top << 16, top & 0xffff0000u);
    } else {
      float x[kVec];
      get(x);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
        if (!finite || bits < 0x7f800000u) top = max(top, bits);
      }
      return top;
    }
  }
  __device__ __forceinline__ void set(const float (&x)[kVec]) {
    if constexpr (kBytes < 4) {
      const __nv_bfloat16 y = __float2bfloat16_rn(x[0]);
      word = *reinterpret_cast<const uint16_t*>(&y);
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(&word);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if constexpr (sizeof(T) == 4) {
          w[i] = __float_as_uint(x[i]);
        } else if (i % 2 == 0) {
          const __nv_bfloat162 y = __floats2bfloat162_rn(x[i], x[i + 1]);
          w[i / 2] = *reinterpret_cast<const uint32_t*>(&y);
        }
      }
    }
  }
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

// Two floats as one operand of the packed multiply-adds.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  return (uint64_t)__float_as_uint(hi) << 32 | __float_as_uint(lo);
}
__device__ __forceinline__ float pair_lo(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float pair_hi(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// The (cos, sin) of a unit's pairs, and where a table of rows in shared memory holds
// them: 16 bytes of two pairs (cos, cos, sin, sin: two-piece units; cos, sin, cos, sin:
// whole pairs in a piece), those of neighbouring units side by side, so that the
// threads of neighbouring units read neighbouring words.
template <int kVec, bool kInter>
struct RotaryTurns {
  static constexpr bool kTwo = RotaryUnits<kVec, kInter>::kTwo;
  static constexpr int kPairs = kTwo ? kVec : kVec / 2;   // of a unit
  float c[kPairs], s[kPairs];

  static __device__ __forceinline__ void put(float* row, int pair, int pairs, float c, float s) {
    if constexpr (kPairs == 1) {
      row[2 * pair] = c;
      row[2 * pair + 1] = s;
    } else {
      const int unit = pair / kPairs, e = pair % kPairs;
      float* at = row + ((e / 2) * (pairs / kPairs) + unit) * 4 + (kTwo ? e % 2 : 2 * (e % 2));
      at[0] = c;
      at[kTwo ? 2 : 1] = s;
    }
  }
  __device__ __forceinline__ void get(const float* row, int pair, int pairs) {
    if constexpr (kPairs == 1) {
      const float2 x = *reinterpret_cast<const float2*>(row + 2 * pair);
      c[0] = x.x, s[0] = x.y;
    } else {
#pragma unroll
      for (int e = 0; e < kPairs; e += 2) {
        const float4 x = *reinterpret_cast<const float4*>(
            row + ((e / 2) * (pairs / kPairs) + pair / kPairs) * 4);
        c[e] = x.x;
        c[e + 1] = kTwo ? x.y : x.z;
        s[e] = kTwo ? x.z : x.y;
        s[e + 1] = x.w;
      }
    }
  }
  // Turns the unit's pieces.
  __device__ __forceinline__ void turn(float (&x)[kVec], float (&y)[kVec]) const {
    if constexpr (kVec == 1) {
      const float a = x[0], b = y[0];
      x[0] = fmaf(a, c[0], -b * s[0]);
      y[0] = fmaf(a, s[0], b * c[0]);
    } else if constexpr (kTwo) {
#pragma unroll
      for (int i = 0; i < kVec; i += 2) {
        const uint64_t a = pair_of(x[i], x[i + 1]), b = pair_of(y[i], y[i + 1]);
        const uint64_t cc = pair_of(c[i], c[i + 1]), ss = pair_of(s[i], s[i + 1]);
        const uint64_t u = pair_fma(a, cc, pair_mul(b, pair_of(-s[i], -s[i + 1])));
        const uint64_t v = pair_fma(a, ss, pair_mul(b, cc));
        x[i] = pair_lo(u), x[i + 1] = pair_hi(u);
        y[i] = pair_lo(v), y[i + 1] = pair_hi(v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVec; i += 2) {
        const float a = x[i], b = x[i + 1];
        x[i] = fmaf(a, c[i / 2], -b * s[i / 2]);
        x[i + 1] = fmaf(a, s[i / 2], b * c[i / 2]);
      }
    }
  }
};

// The table of n rows, 2 * pairs floats each, by kThreads threads; position(row) is a
// row's.  A thread keeps its pair and computes its step once.
template <int kVec, bool kInter, int kThreads, typename Position>
__device__ __forceinline__ void rotary_table(float* table, const double* freq, int pairs,
                                             float magnitude, int n, Position position) {
  if (pairs == 0) return;
  const int each = kThreads / pairs, row0 = threadIdx.x / pairs, pair = threadIdx.x - row0 * pairs;
  if (row0 >= each || row0 >= n) return;
  const RotaryStep step = rotary_step(freq[pair]);
  for (int row = row0; row < n; row += each) {
    const float2 t = rotary_cos_sin(rotary_phase(position(row), step));
    RotaryTurns<kVec, kInter>::put(table + 2 * row * pairs, pair, pairs, t.x * magnitude,
                                   t.y * magnitude);
  }
}

// Turns n rows of `heads` heads: from + row * st + head * sh to to + row * ot + head * oh.
// A thread keeps one unit of one row, whose (cos, sin) it reads once, and goes through
// the heads, kAhead of them in flight.
template <typename T, int kVec, bool kInter, int kThreads>
__device__ __forceinline__ void rotary_rows(const float* table, int pairs, int width, int n,
                                            int heads, const T* from, int64_t st, int64_t sh,
                                            T* to, int64_t ot, int64_t oh) {
  using Units = RotaryUnits<kVec, kInter>;
  using Piece = RotaryPiece<T, kVec>;
  constexpr int kAhead = Units::kTwo ? 4 : 8;
  const int units = Units::count(width, pairs), slots = kThreads / units;
  const int slot = threadIdx.x / units, each = max(1, slots / n);   // threads of a (row, unit)
  const int row0 = slot / each, head0 = slot - row0 * each, rows = slots / each;
  if (row0 >= rows) return;
  const Units unit(threadIdx.x - slot * units, pairs);
  const int second = unit.b - unit.a;
  for (int row = row0; row < n; row += rows) {
    RotaryTurns<kVec, kInter> turns;
    if (unit.pair >= 0) turns.get(table + 2 * row * pairs, unit.pair, pairs);
    const T* src = from + row * st + head0 * sh + unit.a;
    T* dst = to + row * ot + head0 * oh + unit.a;
    const int64_t next = each * sh, next_out = each * oh;
    for (int h = head0; h < heads;) {
      Piece x[kAhead], y[kAhead];
      const int left = (heads - h + each - 1) / each;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (j < left) {
          x[j].load(src);
          if (unit.two()) y[j].load(src + second);
        }
        src += next;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (j < left) {
          if (unit.pair >= 0) {
            float u[kVec], v[kVec];
            x[j].get(u);
            if constexpr (Units::kTwo) y[j].get(v);
            turns.turn(u, v);
            x[j].set(u);
            if constexpr (Units::kTwo) y[j].set(v);
          }
          x[j].store(dst);
          if (unit.two()) y[j].store(dst + second);
        }
        dst += next_out;
      }
      h += each * kAhead;
    }
  }
}

// Out of line, with registers of its own, where it is one call of several.
template <typename T, int kVec, bool kInter, int kThreads>
static __device__ __noinline__ void rotary_rows_apart(const float* table, int pairs, int width,
                                                      int n, int heads, const T* from, int64_t st,
                                                      int64_t sh, T* to, int64_t ot, int64_t oh) {
  rotary_rows<T, kVec, kInter, kThreads>(table, pairs, width, n, heads, from, st, sh, to, ot, oh);
}

// The widest piece that `takes` the layout: calls f with its width (16 bytes, 8, 4, or one
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
    if constexpr (kHalf > 2)
      if (alignment % 4 == 0 && RotaryUnits<2, kInter>::takes(width, pairs))
        return f(std::integral_constant<int, 2>{}, inter);
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
